// Products of 8-bit rows with a quantized matrix (dz_cuda_matmul_q8_async):
//   C[m][n] = T(sum_k a[m][k] level[k][n] * s_a[m] * s_w[n] + bias[n]),
// the sums exact in int32 (K <= 131072 and |a level| <= 128 * 127).
//
// Both operands are read as they are: the rows, and the matrix's signed levels
// in their K-major 16 KB blocks [n / 128][k / 128][n % 128][k % 128].
#include "dz_cuda.h"

#include <atomic>

#include "q8matmul.cuh"
#include "qlevels.cuh"

namespace dz {

// ------------------------------------------------------------- few rows
//
// Bound by the stream of levels. A block of eight warps takes tiles of 16
// columns, each warp every eighth block of 128 rows of W: 2 KB that its lanes
// load 16 bytes at a time straight into the A operands of four 8-bit MMAs
// (m16n8k32, columns as the MMA's rows), the k order within a block being free
// as long as the activations, staged in shared memory, follow it. Four such
// pieces are in flight per warp, across tile borders. The warps' sums meet in
// shared memory once per tile. The next kernel may be launched at once (it waits
// for this one before it touches memory, but for a matrix's levels): a stream of
// 1 x 4096 x 32000 products takes 23.9 us each instead of 25.7.

constexpr int Q8V_WARPS = 8;
constexpr int Q8V_RING = 4;

__device__ __forceinline__ uint4 q8_ldg(const int8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

__device__ __forceinline__ void q8_mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Bytes of a staged row: rows follow each other 64 bytes off a multiple of 128,
// so that the eight 16-byte loads of a quarter warp meet all banks.
__host__ __device__ __forceinline__ int q8v_pitch(int nkb) { return nkb * 128 + 64; }

template <typename T, int G, bool STAGED>    // G groups of 8 rows
__global__ void __launch_bounds__(Q8V_WARPS * 32, 2) dz_q8mv_kernel(const __grid_constant__ Q8MatArgs a) {
    extern __shared__ __align__(16) int8_t q8v_smem[];
    __shared__ int red[2][Q8V_WARPS][G * 8 * 16];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int m0 = blockIdx.y * (G * 8), rows = min(G * 8, a.M - m0);
    const int ntiles = (a.N + 15) >> 4;
    const int first = (int)((long long)ntiles * blockIdx.x / gridDim.x);
    const int last = (int)((long long)ntiles * (blockIdx.x + 1) / gridDim.x);
    const int per = (a.nkb + Q8V_WARPS - 1) / Q8V_WARPS;           // pieces of a tile for each warp
    uint4 ring[Q8V_RING][4];
    int lt = first, lk = warp;               // the next piece to load
    auto load = [&](uint4 (&w)[4]) {
        if (lt >= last) return;
        if (lk < a.nkb) {
            const int8_t* p = a.levels + (((long long)(lt >> 3) * a.nkb + lk) << 14) + ((lt & 7) * 16 + g) * 128 + t * 16;
            w[0] = q8_ldg(p);
            w[1] = q8_ldg(p + 8 * 128);
            w[2] = q8_ldg(p + 64);
            w[3] = q8_ldg(p + 8 * 128 + 64);
        } else {
            w[0] = w[1] = w[2] = w[3] = make_uint4(0, 0, 0, 0);
        }
        lk += Q8V_WARPS;
        if (lk >= per * Q8V_WARPS + warp) {
            lk = warp;
            lt++;
        }
    };
#pragma unroll
    for (int i = 0; i < Q8V_RING; i++) load(ring[i]);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the matrix is no kernel's output, the rows are
    const int8_t* x = a.a + (long long)m0 * a.lda;
    const int kept = (a.K + 15) & ~15;       // <= lda: what lies past K meets levels of 0
    const int pitch = q8v_pitch(a.nkb);
    if (STAGED) {
        const int chunks = a.nkb * 8;
        for (int i = threadIdx.x; i < rows * chunks; i += Q8V_WARPS * 32) {
            const int r = i / chunks, k = (i - r * chunks) * 16;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (k < kept) v = *reinterpret_cast<const uint4*>(x + r * a.lda + k);
            *reinterpret_cast<uint4*>(q8v_smem + r * pitch + k) = v;
        }
        __syncthreads();
    }
    int acc[G][4];
#pragma unroll
    for (int i = 0; i < G; i++) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0;
    int tile = first, piece = 0, buffer = 0;
    const int total = (last - first) * per;
    for (int base = 0; base < total; base += Q8V_RING) {
#pragma unroll
        for (int i = 0; i < Q8V_RING; i++) {
            if (base + i >= total) break;
            const int kb = warp + piece * Q8V_WARPS;
            if (kb < a.nkb) {
#pragma unroll
                for (int q = 0; q < G; q++) {
                    uint4 b0 = make_uint4(0, 0, 0, 0), b1 = b0;
                    if (q * 8 + g < rows) {
                        const int k = kb * 128 + t * 16;
                        if (STAGED) {
                            const int8_t* p = q8v_smem + (q * 8 + g) * pitch + k;
                            b0 = *reinterpret_cast<const uint4*>(p);
                            b1 = *reinterpret_cast<const uint4*>(p + 64);
                        } else {
                            const int8_t* p = x + (q * 8 + g) * a.lda + k;
                            if (k < kept) b0 = *reinterpret_cast<const uint4*>(p);
                            if (k + 64 < kept) b1 = *reinterpret_cast<const uint4*>(p + 64);
                        }
                    }
                    const uint4 (&w)[4] = ring[i];
                    q8_mma(acc[q], w[0].x, w[1].x, w[2].x, w[3].x, b0.x, b1.x);
                    q8_mma(acc[q], w[0].y, w[1].y, w[2].y, w[3].y, b0.y, b1.y);
                    q8_mma(acc[q], w[0].z, w[1].z, w[2].z, w[3].z, b0.z, b1.z);
                    q8_mma(acc[q], w[0].w, w[1].w, w[2].w, w[3].w, b0.w, b1.w);
                }
            }
            load(ring[i]);
            if (++piece < per) continue;
            // the tile's sums: every warp's in shared memory, one barrier, then a thread for each output
            piece = 0;
#pragma unroll
            for (int q = 0; q < G; q++) {
                int* to = red[buffer][warp] + (q * 8 + 2 * t) * 16 + g;
                to[0] = acc[q][0];
                to[16] = acc[q][1];
                to[8] = acc[q][2];
                to[24] = acc[q][3];
                acc[q][0] = acc[q][1] = acc[q][2] = acc[q][3] = 0;
            }
            __syncthreads();
            for (int o = threadIdx.x; o < rows * 16; o += Q8V_WARPS * 32) {
                const int n = tile * 16 + (o & 15), m = m0 + (o >> 4);
                int sum = 0;
#pragma unroll
                for (int w = 0; w < Q8V_WARPS; w++) sum += red[buffer][w][o];
                if (n < a.N)
                    static_cast<T*>(a.c)[m * a.ldc + n] =
                        q8_finish<T>(sum, a.a_scales[m], a.col_scale[n], a.bias ? a.bias[n] : 0.0f);
            }
            buffer ^= 1;                     // the one written two tiles ago has been read by all since the last barrier
            tile++;
        }
    }
}

constexpr int Q8V_SMEM = 96 * 1024;          // staged rows of a block, two blocks to an SM

template <typename T, int G, bool STAGED> static cudaError_t q8mv_g(const Q8MatArgs& a, int device, int sms, cudaStream_t st) {
    static std::atomic<bool> ready[Q8_DEVICES];
    if (STAGED && !ready[device].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(dz_q8mv_kernel<T, G, STAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, Q8V_SMEM);
        if (e != cudaSuccess) return e;
        ready[device].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    const int ntiles = (a.N + 15) / 16;
    cfg.gridDim = dim3((unsigned)(ntiles < 2 * sms ? ntiles : 2 * sms), (unsigned)((a.M + G * 8 - 1) / (G * 8)));
    cfg.blockDim = dim3(Q8V_WARPS * 32);
    cfg.dynamicSmemBytes = STAGED ? (size_t)(a.M < G * 8 ? a.M : G * 8) * q8v_pitch(a.nkb) : 0;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, dz_q8mv_kernel<T, G, STAGED>, a);
}

template <typename T> static cudaError_t q8mv_t(const Q8MatArgs& a, int rows, int device, int sms, cudaStream_t st) {
    if (rows == 16) return q8mv_g<T, 2, true>(a, device, sms, st);
    // rows that fit are staged, others read from L2 with every piece of levels
    if ((size_t)(a.M < 8 ? a.M : 8) * q8v_pitch(a.nkb) <= (size_t)Q8V_SMEM) return q8mv_g<T, 1, true>(a, device, sms, st);
    return q8mv_g<T, 1, false>(a, device, sms, st);
}

static cudaError_t q8mv_launch(const Q8MatArgs& a, int rows, int type, int device, int sms, cudaStream_t st) {
    if (type == DZ_TYPE_F32) return q8mv_t<float>(a, rows, device, sms, st);
    if (type == DZ_TYPE_F16) return q8mv_t<__half>(a, rows, device, sms, st);
    return q8mv_t<__nv_bfloat16>(a, rows, device, sms, st);
}

}  // namespace dz

using namespace dz;

extern "C" int dz_cuda_matmul_q8_async(const int8_t* A, size_t lda, const float* a_scales, const dz_cuda_qmatrix_t* weights,
                                       const float* bias, void* C, size_t ldc, size_t m, size_t k, int type, void* stream) {
    if (!A || !a_scales || !weights || !C) return fail(DZ_E_INVALID, "matmul_q8: null argument");
    QLevels w;
    dz_qmatrix_levels(weights, &w);
    if (!type_ok(type)) return fail(DZ_E_INVALID, "matmul_q8: unknown element type %d", type);
    if (m == 0 || m > (1u << 24) || k != (size_t)w.K)
        return fail(DZ_E_INVALID, "matmul_q8: m must be 1..2^24 and k the matrix rows (%d)", w.K);
    if (w.gran == DZ_GRAN_ROW) return fail(DZ_E_UNSUPPORTED, "matmul_q8: row scales do not factor out of 8-bit rows");
    if (!w.levels) return fail(DZ_E_UNSUPPORTED, "matmul_q8: matrices of more than 131072 rows are not supported");
    if (((uintptr_t)A | lda) & 15) return fail(DZ_E_INVALID, "matmul_q8: rows must start on 16-byte boundaries");
    if (lda < k || lda >= (1ull << 40) || ldc < (size_t)w.N || ldc > (1ull << 40))
        return fail(DZ_E_INVALID, "matmul_q8: row strides must hold k (%zu) and n (%d) elements", k, w.N);
    if ((((uintptr_t)a_scales | (uintptr_t)bias) & 3) || (uintptr_t)C % type_bytes(type))
        return fail(DZ_E_INVALID, "matmul_q8: scales, bias or output are not aligned to their type");
    DeviceGuard g(w.device);
    if (!g.ok) return fail(DZ_E_DEVICE, "cannot select device %d", w.device);
    if (w.device >= Q8_DEVICES) return fail(DZ_E_UNSUPPORTED, "matmul_q8: device ordinals below %d", Q8_DEVICES);
    static std::atomic<int> known[Q8_DEVICES];
    int sms = known[w.device].load(std::memory_order_relaxed);
    if (!sms) {
        DZ_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, w.device));
        known[w.device].store(sms, std::memory_order_relaxed);
    }
    Q8MatArgs a;
    a.a = A;
    a.lda = (long long)lda;
    a.a_scales = a_scales;
    a.levels = w.levels;
    a.col_scale = w.col_scale;
    a.bias = bias;
    a.c = C;
    a.ldc = (long long)ldc;
    a.M = (int)m;
    a.N = w.N;
    a.K = w.K;
    a.nkb = (w.K + 127) / 128;
    const Q8Plan plan = q8_plan(a.M, a.K, a.N, sms, Q8V_SMEM);
    cudaStream_t st = (cudaStream_t)stream;
    DZ_CUDA(plan.rows <= 16 ? q8mv_launch(a, plan.rows, type, w.device, sms, st)
                            : dz_q8gemm_launch(a, w.map, plan, type, w.device, sms, st));
    return DZ_OK;
}
