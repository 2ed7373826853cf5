// Rows in 8 bits (dz_cuda_norm_q8): residual addition, root-mean-square norm
// and quantization in one pass over the rows.
//
// code = round_half_away(u * (127 / P)), u = gain * h, P = max |u|: the norm's
// factor cancels in the codes and stands in the scale alone, so that codes need
// no more than fp32 steps that every evaluation takes alike.
//
// Bound by HBM for many rows (x, residual, sum: 7 bytes an element in 16 bits),
// by latency for few. A row is held in registers between the reduction and the
// codes: by a warp when it is short, by a block of 256 threads up to 32 KB, and
// longer ones are read again.
#include "dz_cuda.h"

#include <cmath>

#include "shim.cuh"

namespace dz {

constexpr int Q8N_THREADS = 256;

struct Q8NormArgs {
    const void *x, *residual;
    void* sum;
    const float* gain;
    int8_t* codes;
    float* scales;
    long long ldx, ldr, lds, ldc, rows;
    int width, norm;
    int wide;                // every typed row starts on a 16-byte boundary, gains too, and codes on an 8-byte one
    double eps64;
};

template <typename T> union Q8Lane {     // 16 bytes of a row
    uint4 q;
    T e[16 / sizeof(T)];
    __device__ Q8Lane() {}
};

// Sum of squares and the largest magnitude (as bits; above 0x7f7fffff it is not
// finite) over the TEAM threads of a row.
template <int TEAM, typename A> __device__ __forceinline__ void q8_reduce(A& sum, unsigned& top) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, off);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
    }
    if (TEAM == 32) return;
    __shared__ A sums[TEAM / 32];
    __shared__ unsigned tops[TEAM / 32];
    if ((threadIdx.x & 31) == 0) {
        sums[threadIdx.x >> 5] = sum;
        tops[threadIdx.x >> 5] = top;
    }
    __syncthreads();
    sum = 0;
    top = 0;
#pragma unroll
    for (int w = 0; w < TEAM / 32; w++) {
        sum += sums[w];
        top = max(top, tops[w]);
    }
    __syncthreads();
}

// What turns a row's u into codes, and its scale.
struct Q8Row {
    float raise, inverse, scale;
    bool empty;              // zeros, or not finite: codes are 0
};

__device__ __forceinline__ Q8Row q8_row(const Q8NormArgs& a, unsigned top, double mean) {
    Q8Row r;
    const float peak = __uint_as_float(top);
    r.raise = top < 0x0D800000u ? 0x1p100f : 1.0f;      // below 2^-100 the inverse would leave fp32
    r.empty = top == 0 || top > 0x7f7fffffu;
    r.inverse = __fdiv_rn(127.0f, peak * r.raise);
    r.scale = __fdiv_rn(peak, 127.0f);
    if (top > 0x7f7fffffu) {
        r.scale = __int_as_float(0x7fc00000);
    } else if (top == 0) {
        r.scale = 0.0f;
    } else if (a.norm) {
        const double m = mean + a.eps64;
        if (m > 1e-30 && m < 1e30) {
            float s = rsqrtf((float)m);
            s = s * fmaf(-0.5f * (float)m * s, s, 1.5f);       // a Newton step
            r.scale = __fdiv_rn(peak * s, 127.0f);
        } else {
            r.scale = (float)((double)peak / sqrt(m) / 127.0);
        }
    }
    return r;
}

__device__ __forceinline__ unsigned q8_code(const Q8Row& r, float u) {
    const float v = __fmul_rn(u * r.raise, r.inverse);         // at most 127 and two roundings: no clamp
    return (unsigned)__float2int_rz(__fadd_rn(v, copysignf(0.5f, v))) & 0xffu;
}

// Sums of squares that leave fp32's range are taken again in 64 bits.
__device__ __forceinline__ bool q8_doubtful(float sum) { return !(sum > 1e-25f && sum < 1e37f); }

template <typename T, int TEAM, int V>
__global__ void __launch_bounds__(Q8N_THREADS) dz_norm_q8_kernel(const __grid_constant__ Q8NormArgs a) {
    constexpr int E = 16 / (int)sizeof(T);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int t = threadIdx.x % TEAM;
    const long long row = (long long)blockIdx.x * (Q8N_THREADS / TEAM) + threadIdx.x / TEAM;
    if (row >= a.rows) return;               // whole teams
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.ldr : nullptr;
    T* out = a.sum ? static_cast<T*>(a.sum) + row * a.lds : nullptr;
    Q8Lane<T> h[V], r[V];
    auto load = [&](const T* in, Q8Lane<T> (&to)[V]) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int at = (j * TEAM + t) * E;
            if (a.wide && at + E <= a.width) {
                to[j].q = *reinterpret_cast<const uint4*>(in + at);
            } else {
#pragma unroll
                for (int i = 0; i < E; i++) to[j].e[i] = at + i < a.width ? in[at + i] : dz_from_float<T>(0.0f);
            }
        }
    };
    load(x, h);
    if (res) {
        load(res, r);
#pragma unroll
        for (int j = 0; j < V; j++)
#pragma unroll
            for (int i = 0; i < E; i++) h[j].e[i] = dz_from_float<T>(dz_to_float(h[j].e[i]) + dz_to_float(r[j].e[i]));
    }
    if (out) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int at = (j * TEAM + t) * E;
            if (a.wide && at + E <= a.width) {
                *reinterpret_cast<uint4*>(out + at) = h[j].q;
            } else {
#pragma unroll
                for (int i = 0; i < E; i++)
                    if (at + i < a.width) out[at + i] = h[j].e[i];
            }
        }
    }
    // the gains of E elements at `at`
    auto gains = [&](int at, float (&g)[E]) {
        if (!a.gain) {
#pragma unroll
            for (int i = 0; i < E; i++) g[i] = 1.0f;
        } else if (a.wide && at + E <= a.width) {
#pragma unroll
            for (int i = 0; i < E; i += 4) {
                const float4 v = *reinterpret_cast<const float4*>(a.gain + at + i);
                g[i] = v.x;
                g[i + 1] = v.y;
                g[i + 2] = v.z;
                g[i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < E; i++) g[i] = at + i < a.width ? a.gain[at + i] : 0.0f;
        }
    };
    float sum = 0.0f;
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < V; j++) {
        float g[E];
        gains((j * TEAM + t) * E, g);
#pragma unroll
        for (int i = 0; i < E; i++) {
            const float v = dz_to_float(h[j].e[i]);
            sum = fmaf(v, v, sum);
            top = max(top, __float_as_uint(__fmul_rn(g[i], v)) & 0x7fffffffu);
        }
    }
    q8_reduce<TEAM>(sum, top);
    double mean = (double)sum / a.width;
    if (a.norm && q8_doubtful(sum)) {        // the whole team alike
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < V; j++)
#pragma unroll
            for (int i = 0; i < E; i++) s += (double)dz_to_float(h[j].e[i]) * (double)dz_to_float(h[j].e[i]);
        unsigned same = top;
        q8_reduce<TEAM>(s, same);
        mean = s / a.width;
    }
    const Q8Row k = q8_row(a, top, mean);
    int8_t* codes = a.codes + row * a.ldc;
#pragma unroll
    for (int j = 0; j < V; j++) {
        const int at = (j * TEAM + t) * E;
        if (at >= a.width) break;
        float g[E];
        gains(at, g);
        unsigned word[E / 4];
#pragma unroll
        for (int i = 0; i < E; i++) {
            const unsigned c = k.empty ? 0u : q8_code(k, __fmul_rn(g[i], dz_to_float(h[j].e[i])));
            word[i / 4] = i % 4 ? word[i / 4] | c << (i % 4 * 8) : c;
        }
        if (a.wide && at + E <= a.width) {
            if (E == 8)
                *reinterpret_cast<uint2*>(codes + at) = make_uint2(word[0], word[E / 4 - 1]);
            else
                *reinterpret_cast<unsigned*>(codes + at) = word[0];
        } else {
#pragma unroll
            for (int i = 0; i < E; i++)
                if (at + i < a.width) codes[at + i] = (int8_t)(word[i / 4] >> (i % 4 * 8));
        }
    }
    if (t == 0) a.scales[row] = k.scale;
}

// Rows of any width, read again for their codes.
template <typename T> __global__ void __launch_bounds__(Q8N_THREADS) dz_norm_q8_long_kernel(const __grid_constant__ Q8NormArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.ldr : nullptr;
    T* out = a.sum ? static_cast<T*>(a.sum) + row * a.lds : nullptr;
    auto value = [&](int i) { return res ? dz_from_float<T>(dz_to_float(x[i]) + dz_to_float(res[i])) : x[i]; };
    double sum = 0.0;
    unsigned top = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < a.width; i += Q8N_THREADS) {
        const T h = value(i);
        const float v = dz_to_float(h);
        if (out) out[i] = h;                 // the same thread reads it below
        sum += (double)v * (double)v;
        top = max(top, __float_as_uint(a.gain ? __fmul_rn(a.gain[i], v) : v) & 0x7fffffffu);
    }
    q8_reduce<Q8N_THREADS>(sum, top);
    const Q8Row k = q8_row(a, top, sum / a.width);
    int8_t* codes = a.codes + row * a.ldc;
#pragma unroll 4
    for (int i = threadIdx.x; i < a.width; i += Q8N_THREADS) {
        const float v = dz_to_float(out ? out[i] : value(i));
        codes[i] = k.empty ? (int8_t)0 : (int8_t)q8_code(k, a.gain ? __fmul_rn(a.gain[i], v) : v);
    }
    if (threadIdx.x == 0) a.scales[row] = k.scale;
}

template <typename T> static cudaError_t q8_norm_t(const Q8NormArgs& a, cudaStream_t st) {
    constexpr int E = 16 / (int)sizeof(T);
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(Q8N_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const int vectors = (a.width + E - 1) / E;
    cfg.gridDim = dim3((unsigned)(vectors <= 64 ? (a.rows + Q8N_THREADS / 32 - 1) / (Q8N_THREADS / 32) : a.rows));
    if (vectors <= 32) return cudaLaunchKernelEx(&cfg, dz_norm_q8_kernel<T, 32, 1>, a);
    if (vectors <= 64) return cudaLaunchKernelEx(&cfg, dz_norm_q8_kernel<T, 32, 2>, a);
    if (vectors <= 256) return cudaLaunchKernelEx(&cfg, dz_norm_q8_kernel<T, 256, 1>, a);
    if (vectors <= 512) return cudaLaunchKernelEx(&cfg, dz_norm_q8_kernel<T, 256, 2>, a);
    if (vectors <= 1024) return cudaLaunchKernelEx(&cfg, dz_norm_q8_kernel<T, 256, 4>, a);
    if (vectors <= 2048) return cudaLaunchKernelEx(&cfg, dz_norm_q8_kernel<T, 256, 8>, a);
    return cudaLaunchKernelEx(&cfg, dz_norm_q8_long_kernel<T>, a);
}

}  // namespace dz

using namespace dz;

static int q8_operand(const char* what, const void* base, size_t stride, size_t width, int type) {
    if ((uintptr_t)base % type_bytes(type)) return fail(DZ_E_INVALID, "norm_q8: %s is not aligned to its type", what);
    if (stride < width || stride > (1ull << 40))
        return fail(DZ_E_INVALID, "norm_q8: %s rows of %zu elements do not hold %zu", what, stride, width);
    return DZ_OK;
}

extern "C" int dz_cuda_norm_q8(const dz_norm_q8_t* p, size_t rows, size_t width, void* stream) {
    if (!p || !p->x || !p->codes || !p->scales) return fail(DZ_E_INVALID, "norm_q8: null argument");
    if (!type_ok(p->type)) return fail(DZ_E_INVALID, "norm_q8: unknown element type %d", p->type);
    if (rows == 0 || rows > (size_t)INT32_MAX || width == 0 || width > ((size_t)1 << 30))
        return fail(DZ_E_INVALID, "norm_q8: rows must be 1..2^31-1 and width 1..2^30");
    int rc = q8_operand("x", p->x, p->x_stride, width, p->type);
    if (!rc && p->residual) rc = q8_operand("residual", p->residual, p->residual_stride, width, p->type);
    if (!rc && p->sum_out) rc = q8_operand("sum_out", p->sum_out, p->sum_stride, width, p->type);
    if (rc) return rc;
    if (p->codes_stride < width || p->codes_stride > (1ull << 40))
        return fail(DZ_E_INVALID, "norm_q8: rows of %zu codes do not hold %zu", p->codes_stride, width);
    if (((uintptr_t)p->gain | (uintptr_t)p->scales) & 3) return fail(DZ_E_INVALID, "norm_q8: gains or scales are not aligned");
    if (p->norm != 0 && p->norm != 1) return fail(DZ_E_INVALID, "norm_q8: norm must be 0 or 1");
    if (p->norm && !(p->eps >= 0.0 && std::isfinite(p->eps)))
        return fail(DZ_E_INVALID, "norm_q8: eps must be finite and >= 0");
    DeviceGuard g(p->device);
    if (!g.ok) return fail(DZ_E_DEVICE, "cannot select device %d", p->device);
    Q8NormArgs a;
    a.x = p->x;
    a.residual = p->residual;
    a.sum = p->sum_out;
    a.gain = p->gain;
    a.codes = p->codes;
    a.scales = p->scales;
    a.ldx = (long long)p->x_stride;
    a.ldr = p->residual ? (long long)p->residual_stride : 0;
    a.lds = p->sum_out ? (long long)p->sum_stride : 0;
    a.ldc = (long long)p->codes_stride;
    a.rows = (long long)rows;
    a.width = (int)width;
    a.norm = p->norm;
    a.eps64 = p->norm ? p->eps : 0.0;
    const uintptr_t bases = (uintptr_t)p->x | (uintptr_t)p->residual | (uintptr_t)p->sum_out | (uintptr_t)p->gain;
    a.wide = bases % 16 == 0 && (a.ldx | a.ldr | a.lds) * (long long)type_bytes(p->type) % 16 == 0 &&
             ((uintptr_t)p->codes | (uintptr_t)a.ldc) % 8 == 0;
    cudaStream_t st = (cudaStream_t)stream;
    DZ_CUDA(p->type == DZ_TYPE_F32   ? q8_norm_t<float>(a, st)
            : p->type == DZ_TYPE_F16 ? q8_norm_t<__half>(a, st)
                                     : q8_norm_t<__nv_bfloat16>(a, st));
    return DZ_OK;
}
