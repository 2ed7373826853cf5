// Group-scaled 4-bit products: the device layout, the kernel (gmatvec.cuh) and
// the C entry points, in a translation unit of their own.
#include "dz_cuda.h"

#include <cmath>
#include <new>

#include "gmatvec.cuh"
#include "shim.cuh"

namespace dz {

__device__ __forceinline__ int gmv_code(const uint8_t* packed, long long i) {
    return (packed[i >> 1] >> ((i & 1) * 4)) & 15;
}

// One thread per word of the records' codes. `bad` is set for a code of 15.
__global__ void dz_gmv_repack_kernel(const uint8_t* __restrict__ packed, GmvMatrix w, int* __restrict__ bad) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const long long total = (long long)w.ntiles * w.nblocks * (GMV_CODES / 4);
    if (i >= total) return;
    const int word = (int)(i % (GMV_CODES / 4));
    const long long r = i / (GMV_CODES / 4);
    const int half = word >> 7, lane = (word >> 2) & 31, q = word & 3;
    const int g = lane >> 2, t = lane & 3;
    const int n = (int)(r / w.nblocks) * GMV_TILE + g + 8 * (q & 1);
    const int k0 = (int)(r % w.nblocks) * GMV_BLOCK + 64 * half + 32 * (q >> 1) + 8 * t;
    uint32_t v = 0;
    if (n < w.N) {
        for (int j = 0; j < 8; j++) {
            const int k = k0 + j;
            if (k >= w.K) break;
            const int c = gmv_code(packed, (long long)k * w.N + n);
            if (c > 14) *bad = 1;
            const uint32_t level = (uint32_t)(c - 7) & 15u;
            v |= level << (j < 4 ? 8 * j + 4 : 8 * (j - 4));
        }
    }
    *reinterpret_cast<uint32_t*>(w.rec + r * w.rec_bytes + 4 * word) = v;
}

// One thread per scale slot of the records. `bad` is set for a scale that is
// negative or not finite.
template <typename S>
__global__ void dz_gmv_scales_kernel(const S* __restrict__ scales, GmvMatrix w, int* __restrict__ bad) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int per = GMV_BLOCK / w.group * GMV_TILE;
    if (i >= (long long)w.ntiles * w.nblocks * per) return;
    const int at = (int)(i % per);
    const long long r = i / per;
    const int n = (int)(r / w.nblocks) * GMV_TILE + at % GMV_TILE;
    const int k = (int)(r % w.nblocks) * GMV_BLOCK + at / GMV_TILE * w.group;
    S s = dz_from_float<S>(0.0f);
    if (n < w.N && k < w.K) {
        s = scales[(long long)(k / w.group) * w.N + n];
        const float f = dz_to_float(s);
        if (!(f >= 0.0f && f <= 3.402823466e38f)) *bad = 2;
    }
    reinterpret_cast<S*>(w.rec + r * w.rec_bytes + GMV_CODES)[at] = s;
}

// One thread per element: dst = scale * level.
template <typename S> __global__ void dz_gmv_dequant_kernel(GmvMatrix w, float* __restrict__ dst) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (long long)w.K * w.N) return;
    const int k = (int)(i / w.N), n = (int)(i % w.N);
    const uint8_t* rec = w.rec + ((long long)(n / GMV_TILE) * w.nblocks + k / GMV_BLOCK) * w.rec_bytes;
    const int kk = k % GMV_BLOCK, j = kk & 7, c = n % GMV_TILE;
    const int word = (kk >> 6) * 128 + ((c & 7) * 4 + ((kk >> 3) & 3)) * 4 + 2 * ((kk >> 5) & 1) + (c >> 3);
    const int byte = rec[4 * word + (j & 3)];
    const int level = (int)((uint32_t)(j < 4 ? byte >> 4 : byte & 15) << 28) >> 28;
    dst[i] = dz_to_float(reinterpret_cast<const S*>(rec + GMV_CODES)[kk / w.group * GMV_TILE + c]) * (float)level;
}

// One block per (tile, row): thread (p, c) sums column c over the groups p,
// p + 16, ... in fp32; the 16 parts add in order in shared memory.
template <typename T, typename S> __global__ void __launch_bounds__(256) dz_gmv_simple_kernel(GmvArgs a) {
    __shared__ float part[16][GMV_TILE];
    const GmvMatrix& w = a.w;
    const int c = threadIdx.x % GMV_TILE, p = threadIdx.x / GMV_TILE, m = blockIdx.y;
    const T* x = static_cast<const T*>(a.x) + (long long)m * a.ldx;
    float acc = 0.0f;
    for (int k0 = p * w.group; k0 < w.K; k0 += 16 * w.group) {
        const uint8_t* rec = w.rec + ((long long)blockIdx.x * w.nblocks + k0 / GMV_BLOCK) * w.rec_bytes;
        float s = 0.0f;
        for (int k = k0; k < min(k0 + w.group, w.K); k++) {
            const int kk = k % GMV_BLOCK, j = kk & 7;
            const int word = (kk >> 6) * 128 + ((c & 7) * 4 + ((kk >> 3) & 3)) * 4 + 2 * ((kk >> 5) & 1) + (c >> 3);
            const int byte = rec[4 * word + (j & 3)];
            const int level = (int)((uint32_t)(j < 4 ? byte >> 4 : byte & 15) << 28) >> 28;
            const float v = dz_to_float(x[k]);   // v - v: NaN for an infinity
            s = fmaf((float)level, v, s) + (v - v);
        }
        acc = fmaf(s, dz_to_float(reinterpret_cast<const S*>(rec + GMV_CODES)[k0 % GMV_BLOCK / w.group * GMV_TILE + c]),
                   acc);
    }
    part[p][c] = acc;
    __syncthreads();
    const int n = blockIdx.x * GMV_TILE + c;
    if (p == 0 && n < w.N) {
        float s = 0.0f;
        for (int i = 0; i < 16; i++) s += part[i][c];
        static_cast<T*>(a.y)[(long long)m * a.ldy + n] = dz_from_float<T>(s);
    }
}

template <typename T> static void gmv_launch_t(const GmvArgs& a, dim3 grid, cudaStream_t st) {
    if (a.w.scale_f16)
        dz_gmv_simple_kernel<T, __half><<<grid, 256, 0, st>>>(a);
    else
        dz_gmv_simple_kernel<T, float><<<grid, 256, 0, st>>>(a);
}

cudaError_t dz_gmv_launch(const GmvArgs& a, int, cudaStream_t st) {
    GmvArgs b = a;
    for (int m = 0; m < a.M; m += 65535) {
        b.M = a.M - m < 65535 ? a.M - m : 65535;
        b.x = static_cast<const uint8_t*>(a.x) + (long long)m * a.ldx * type_bytes(a.type);
        b.y = static_cast<uint8_t*>(a.y) + (long long)m * a.ldy * type_bytes(a.type);
        const dim3 grid((unsigned)a.w.ntiles, (unsigned)b.M);
        if (a.type == DZ_TYPE_F32)
            gmv_launch_t<float>(b, grid, st);
        else if (a.type == DZ_TYPE_F16)
            gmv_launch_t<__half>(b, grid, st);
        else
            gmv_launch_t<__nv_bfloat16>(b, grid, st);
    }
    return cudaGetLastError();
}

}  // namespace dz

using namespace dz;

struct dz_cuda_gmatrix {
    int device;
    GmvMatrix m;
};

// K and N up to 2^24 and at most 2^31 records keep the kernels' indexes in range.
constexpr size_t GMV_MAX_DIM = (size_t)1 << 24;

static int gmv_check(const dz_grouped_blob_t* w) {
    if (!w || !w->packed || !w->scales) return fail(DZ_E_INVALID, "gmatrix: null argument");
    if (w->rows == 0 || w->cols == 0 || w->rows > GMV_MAX_DIM || w->cols > GMV_MAX_DIM)
        return fail(DZ_E_INVALID, "gmatrix: rows and cols must be 1..%zu", GMV_MAX_DIM);
    if (w->group != 32 && w->group != 64 && w->group != 128)
        return fail(DZ_E_INVALID, "gmatrix: groups hold 32, 64 or 128 rows, not %zu", w->group);
    if (w->scale_type != DZ_TYPE_F32 && w->scale_type != DZ_TYPE_F16)
        return fail(DZ_E_INVALID, "gmatrix: scales are fp32 or fp16");
    if (w->packed_size != (w->rows * w->cols + 1) / 2 || w->scale_count != ((w->rows - 1) / w->group + 1) * w->cols)
        return fail(DZ_E_INVALID, "gmatrix: %zu code bytes and %zu scales do not fit %zu x %zu in groups of %zu",
                    w->packed_size, w->scale_count, w->rows, w->cols, w->group);
    return DZ_OK;
}

// Lays w out into m->rec on the current device; the staging copies live here.
static int gmv_fill(const dz_grouped_blob_t* w, GmvMatrix* m, cudaStream_t st, uint8_t** codes, uint8_t** scales,
                    int** bad) {
    const size_t sb = w->scale_count * (m->scale_f16 ? 2 : 4);
    const long long recs = (long long)m->ntiles * m->nblocks;
    DZ_CUDA(cudaMalloc(&m->rec, (size_t)recs * m->rec_bytes));
    DZ_CUDA(cudaMalloc(codes, w->packed_size));
    DZ_CUDA(cudaMalloc(scales, sb));
    DZ_CUDA(cudaMalloc(bad, 4));
    // sources in device memory may still be written by any stream
    for (const void* src : {(const void*)w->packed, w->scales}) {
        cudaPointerAttributes at;
        if (cudaPointerGetAttributes(&at, src) != cudaSuccess)
            (void)cudaGetLastError();
        else if (at.type == cudaMemoryTypeDevice || at.type == cudaMemoryTypeManaged) {
            DZ_CUDA(cudaDeviceSynchronize());
            break;
        }
    }
    DZ_CUDA(cudaMemcpyAsync(*codes, w->packed, w->packed_size, cudaMemcpyDefault, st));
    DZ_CUDA(cudaMemcpyAsync(*scales, w->scales, sb, cudaMemcpyDefault, st));
    DZ_CUDA(cudaMemsetAsync(*bad, 0, 4, st));
    const long long words = recs * (GMV_CODES / 4), slots = recs * (GMV_BLOCK / m->group * GMV_TILE);
    dz_gmv_repack_kernel<<<(unsigned)((words + 255) / 256), 256, 0, st>>>(*codes, *m, *bad);
    if (m->scale_f16)
        dz_gmv_scales_kernel<<<(unsigned)((slots + 255) / 256), 256, 0, st>>>((const __half*)*scales, *m, *bad);
    else
        dz_gmv_scales_kernel<<<(unsigned)((slots + 255) / 256), 256, 0, st>>>((const float*)*scales, *m, *bad);
    DZ_CUDA(cudaGetLastError());
    int why = 0;
    DZ_CUDA(cudaMemcpyAsync(&why, *bad, 4, cudaMemcpyDeviceToHost, st));
    DZ_CUDA(cudaStreamSynchronize(st));
    if (why) return fail(DZ_E_INVALID, why == 1 ? "gmatrix: a code of 15" : "gmatrix: a negative or non-finite scale");
    return DZ_OK;
}

extern "C" int dz_cuda_gmatrix_create(int device, const dz_grouped_blob_t* w, dz_cuda_gmatrix_t** out) {
    if (!out) return fail(DZ_E_INVALID, "null output handle");
    *out = nullptr;
    int rc = gmv_check(w);
    if (rc) return rc;
    DeviceGuard g(device);
    if (!g.ok) return fail(DZ_E_DEVICE, "cannot select device %d", device);
    GmvMatrix m;
    m.K = (int)w->rows;
    m.N = (int)w->cols;
    m.group = (int)w->group;
    m.scale_f16 = w->scale_type == DZ_TYPE_F16;
    m.ntiles = (m.N + GMV_TILE - 1) / GMV_TILE;
    m.nblocks = (m.K + GMV_BLOCK - 1) / GMV_BLOCK;
    m.rec_bytes = GMV_CODES + GMV_BLOCK / m.group * GMV_TILE * (m.scale_f16 ? 2 : 4);
    if ((long long)m.ntiles * m.nblocks > (1LL << 30)) return fail(DZ_E_UNSUPPORTED, "gmatrix: too many weights");
    auto* q = new (std::nothrow) dz_cuda_gmatrix;
    if (!q) return fail(DZ_E_NOMEM, "host allocation");
    cudaStream_t st = nullptr;
    uint8_t *codes = nullptr, *scales = nullptr;
    int* bad = nullptr;
    if (cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking) != cudaSuccess)
        rc = fail(DZ_E_DEVICE, "stream creation failed");
    if (!rc) rc = gmv_fill(w, &m, st, &codes, &scales, &bad);
    cudaFree(codes);
    cudaFree(scales);
    cudaFree(bad);
    if (st) cudaStreamDestroy(st);
    if (rc) {
        cudaFree(m.rec);
        delete q;
        return rc;
    }
    q->device = device;
    q->m = m;
    *out = q;
    return DZ_OK;
}

extern "C" void dz_cuda_gmatrix_free(dz_cuda_gmatrix_t* q) {
    if (!q) return;
    DeviceGuard g(q->device);
    cudaFree(q->m.rec);
    delete q;
}

extern "C" size_t dz_cuda_gmatrix_bytes(const dz_cuda_gmatrix_t* q) {
    return q ? (size_t)q->m.ntiles * q->m.nblocks * q->m.rec_bytes : 0;
}

extern "C" int dz_cuda_gmatrix_unpack(const dz_cuda_gmatrix_t* q, float* dst) {
    if (!q || !dst) return fail(DZ_E_INVALID, "null argument");
    DeviceGuard g(q->device);
    const long long total = (long long)q->m.K * q->m.N;
    float* d = nullptr;
    DZ_CUDA(cudaMalloc(&d, total * 4));
    const unsigned grid = (unsigned)((total + 255) / 256);
    if (q->m.scale_f16)
        dz_gmv_dequant_kernel<__half><<<grid, 256>>>(q->m, d);
    else
        dz_gmv_dequant_kernel<float><<<grid, 256>>>(q->m, d);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaMemcpy(dst, d, total * 4, cudaMemcpyDeviceToHost);
    cudaFree(d);
    if (e != cudaSuccess) return fail(DZ_E_DEVICE, "unpack: %s", cudaGetErrorString(e));
    return DZ_OK;
}

extern "C" int dz_cuda_matmul_grouped_async(const void* A, size_t lda, const dz_cuda_gmatrix_t* q, void* C, size_t ldc,
                                            size_t m, size_t k, int type, void* stream) {
    if (!q || !A || !C) return fail(DZ_E_INVALID, "matmul_grouped: null argument");
    if (!type_ok(type)) return fail(DZ_E_INVALID, "matmul_grouped: unknown element type %d", type);
    if (m == 0 || m > (1u << 24) || k != (size_t)q->m.K)
        return fail(DZ_E_INVALID, "matmul_grouped: k must equal the matrix rows, m be 1..%u", 1u << 24);
    if (lda < k || ldc < (size_t)q->m.N || lda > (1ull << 40) || ldc > (1ull << 40))
        return fail(DZ_E_INVALID, "matmul_grouped: row strides must hold a row");
    if (((uintptr_t)A | (uintptr_t)C) % type_bytes(type))
        return fail(DZ_E_INVALID, "matmul_grouped: A and C must be aligned to their element type");
    DeviceGuard g(q->device);
    if (!g.ok) return fail(DZ_E_DEVICE, "cannot select device %d", q->device);
    GmvArgs a;
    a.w = q->m;
    a.x = A;
    a.y = C;
    a.ldx = (long long)lda;
    a.ldy = (long long)ldc;
    a.M = (int)m;
    a.type = type;
    DZ_CUDA(dz_gmv_launch(a, q->device, (cudaStream_t)stream));
    return DZ_OK;
}

extern "C" int dz_cuda_matmul_grouped(const float* A, const dz_cuda_gmatrix_t* q, float* C, size_t m, size_t k) {
    if (!q || !A || !C || m == 0 || m > (1u << 24) || k != (size_t)q->m.K)
        return fail(DZ_E_INVALID, "matmul_grouped: bad arguments (k must equal the matrix rows)");
    DeviceGuard g(q->device);
    const size_t n = (size_t)q->m.N;
    float *dA = nullptr, *dC = nullptr;
    DZ_CUDA(cudaMalloc(&dA, m * k * 4));
    if (cudaMalloc(&dC, m * n * 4) != cudaSuccess) {
        cudaFree(dA);
        return fail(DZ_E_NOMEM, "device allocation");
    }
    cudaError_t e = cudaMemcpy(dA, A, m * k * 4, cudaMemcpyHostToDevice);
    int rc = DZ_OK;
    if (e == cudaSuccess) rc = dz_cuda_matmul_grouped_async(dA, k, q, dC, n, m, k, DZ_TYPE_F32, nullptr);
    if (e == cudaSuccess && rc == DZ_OK) e = cudaMemcpy(C, dC, m * n * 4, cudaMemcpyDeviceToHost);
    cudaFree(dA);
    cudaFree(dC);
    if (rc) return rc;
    if (e != cudaSuccess) return fail(DZ_E_DEVICE, "matmul_grouped: %s", cudaGetErrorString(e));
    return DZ_OK;
}
