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
// longer ones are read again. Blocks stay: the next rows are on their way into
// shared memory while one is worked on (each thread copies what it reads itself,
// so that no barrier is needed; a row ahead in registers took 45 us for 8192 x
// 4096 in bf16, none 54), and the gains of rows up to 8 KB stay in registers.
#include "dz_cuda.h"

#include <atomic>
#include <cmath>

#include "shim.cuh"

namespace dz {

constexpr int Q8N_THREADS = 256;
constexpr int Q8N_DEVICES = 64;    // devices whose launch state is kept

struct Q8NormArgs {
    const void *x, *residual;
    void* sum;
    const float* gain;
    int8_t* codes;
    float* scales;
    long long ldx, ldr, lds, ldc, rows;
    int width, norm;
    double eps64;
};

template <typename T> union Q8Lane {     // 16 bytes of a row
    uint4 q;
    T e[16 / sizeof(T)];
    __device__ Q8Lane() {}
};

// The larger magnitude; a NaN stays one.
__device__ __forceinline__ float q8_larger(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}

// Sum of squares and the largest magnitude over the TEAM threads of a row.
// `turn` alternates from call to call: a place is written again only after a
// barrier that followed its reads.
template <int TEAM, typename A> __device__ __forceinline__ void q8_reduce(A& sum, float& top, int turn) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, off);
        top = q8_larger(top, __shfl_xor_sync(0xffffffffu, top, off));
    }
    if (TEAM == 32) return;
    __shared__ A sums[2][TEAM / 32];
    __shared__ float tops[2][TEAM / 32];
    if ((threadIdx.x & 31) == 0) {
        sums[turn][threadIdx.x >> 5] = sum;
        tops[turn][threadIdx.x >> 5] = top;
    }
    __syncthreads();
    sum = 0;
    top = 0.0f;
#pragma unroll
    for (int w = 0; w < TEAM / 32; w++) {
        sum += sums[turn][w];
        top = q8_larger(top, tops[turn][w]);
    }
}

// What turns a row's u into codes.
struct Q8Row {
    float raise, inverse;
    bool plain;              // raise is 1, and there are codes
    bool empty;              // zeros, or not finite: codes are 0
};

__device__ __forceinline__ Q8Row q8_row(float peak) {
    Q8Row r;
    r.plain = peak >= 0x1p-100f && peak <= 3.402823466e38f;
    r.raise = r.plain ? 1.0f : 0x1p100f;      // below 2^-100 the inverse would leave fp32
    r.empty = !(peak > 0.0f && peak <= 3.402823466e38f);
    r.inverse = __fdiv_rn(127.0f, peak * r.raise);
    return r;
}

__device__ __forceinline__ float q8_scale(const Q8NormArgs& a, float peak, double mean) {
    if (!(peak <= 3.402823466e38f)) return __int_as_float(0x7fc00000);
    if (peak == 0.0f) return 0.0f;
    if (!a.norm) return __fdiv_rn(peak, 127.0f);
    const double m = mean + a.eps64;
    // the reciprocal root is below 1e15 there, and its product with the peak within fp32
    if (!(m > 1e-30 && m < 1e30 && peak < 1e22f)) return (float)((double)peak / sqrt(m) / 127.0);
    float s = rsqrtf((float)m);
    s = s * fmaf(-0.5f * (float)m * s, s, 1.5f);               // a Newton step
    return __fdiv_rn(peak * s, 127.0f);
}

// At most 127 and two roundings before it is rounded: no clamp.
__device__ __forceinline__ int q8_round(float v) { return __float2int_rz(__fadd_rn(v, copysignf(0.5f, v))); }
__device__ __forceinline__ int q8_code(const Q8Row& r, float u) {
    return r.plain ? q8_round(__fmul_rn(u, r.inverse)) : r.empty ? 0 : q8_round(__fmul_rn(u * r.raise, r.inverse));
}

// Sums of squares that leave fp32's range are taken again in 64 bits.
__device__ __forceinline__ bool q8_doubtful(float sum) { return !(sum > 1e-25f && sum < 1e37f); }

// WIDE: rows are whole numbers of 16 bytes and start on such a boundary, gains
// too, and codes on an 8-byte one. A thread then has E elements side by side V
// times and its rows come through shared memory, else each of them TEAM further
// on, loaded as they are needed.
template <int V> struct Q8Ring {
    static constexpr int ROWS = V <= 2 ? 4 : V == 4 ? 3 : 2;         // of a team, in turn
    static constexpr int PART = V * Q8N_THREADS * 16;                // x or the residual of the teams' rows
    static constexpr int BLOCKS = V <= 2 ? 3 : V == 4 ? 2 : 1;       // of an SM
    static constexpr int SMEM = ROWS * 2 * PART;
};

template <typename T, int TEAM, int V, bool WIDE>
__global__ void __launch_bounds__(Q8N_THREADS, Q8Ring<V>::BLOCKS) dz_norm_q8_kernel(const __grid_constant__ Q8NormArgs a) {
    constexpr int E = 16 / (int)sizeof(T);
    constexpr bool KEPT = V * E <= 16;       // gains stay in registers
    extern __shared__ __align__(16) uint8_t q8n_ring[];
    const int t = threadIdx.x % TEAM;
    long long row = (long long)blockIdx.x * (Q8N_THREADS / TEAM) + threadIdx.x / TEAM;
    const long long step = (long long)gridDim.x * (Q8N_THREADS / TEAM);
    // a product that follows may fetch its levels now (it waits for this kernel's end before it reads rows)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (row >= a.rows) return;               // whole teams
    auto place = [&](int j, int i) { return WIDE ? (j * TEAM + t) * E + i : (j * E + i) * TEAM + t; };
    auto load = [&](const void* base, long long ld, Q8Lane<T> (&to)[V]) {
        const T* in = static_cast<const T*>(base) + row * ld;
#pragma unroll
        for (int j = 0; j < V; j++)
#pragma unroll
            for (int i = 0; i < E; i++) to[j].e[i] = place(j, i) < a.width ? in[place(j, i)] : dz_from_float<T>(0.0f);
    };
    // this thread's place in a slot's part, vector j
    auto slot_of = [&](int slot, int part, int j) {
        return q8n_ring + (slot * 2 + part) * Q8Ring<V>::PART + (j * Q8N_THREADS + (int)threadIdx.x) * 16;
    };
    auto copy = [&](int slot, long long r) {
        if (r < a.rows) {
#pragma unroll
            for (int part = 0; part < 2; part++) {
                const T* base = static_cast<const T*>(part ? a.residual : a.x);
                if (!base) continue;
                base += r * (part ? a.ldr : a.ldx);
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (place(j, 0) < a.width)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(slot_of(slot, part, j))),
                                     "l"(base + place(j, 0))
                                     : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto gains = [&](int j, float (&g)[E]) {
        if (!a.gain) {
#pragma unroll
            for (int i = 0; i < E; i++) g[i] = 1.0f;
        } else if (WIDE) {
#pragma unroll
            for (int i = 0; i < E; i += 4) {
                const float4 v = place(j, 0) < a.width ? *reinterpret_cast<const float4*>(a.gain + place(j, i))
                                                       : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                g[i] = v.x;
                g[i + 1] = v.y;
                g[i + 2] = v.z;
                g[i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < E; i++) g[i] = place(j, i) < a.width ? a.gain[place(j, i)] : 0.0f;
        }
    };
    constexpr int AHEAD = Q8Ring<V>::ROWS - 1;
    if (WIDE) {
#pragma unroll
        for (int s = 0; s < AHEAD; s++) copy(s, row + s * step);
    }
    float kept[KEPT ? V : 1][E];
    if (KEPT) {
#pragma unroll
        for (int j = 0; j < V; j++) gains(j, kept[KEPT ? j : 0]);
    }
    int slot = 0;
    for (int turn = 0;; turn ^= 1) {
        Q8Lane<T> h[V];
        if (WIDE) {
            copy(slot + AHEAD >= Q8Ring<V>::ROWS ? slot + AHEAD - Q8Ring<V>::ROWS : slot + AHEAD, row + AHEAD * step);
            asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD) : "memory");
#pragma unroll
            for (int j = 0; j < V; j++) {
                h[j].q = place(j, 0) < a.width ? *reinterpret_cast<const uint4*>(slot_of(slot, 0, j)) : make_uint4(0, 0, 0, 0);
                if (a.residual) {
                    Q8Lane<T> r;
                    r.q = place(j, 0) < a.width ? *reinterpret_cast<const uint4*>(slot_of(slot, 1, j)) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < E; i++) h[j].e[i] = dz_from_float<T>(dz_to_float(h[j].e[i]) + dz_to_float(r.e[i]));
                }
            }
            slot = slot + 1 == Q8Ring<V>::ROWS ? 0 : slot + 1;
        } else {
            load(a.x, a.ldx, h);
            if (a.residual) {
                Q8Lane<T> r[V];
                load(a.residual, a.ldr, r);
#pragma unroll
                for (int j = 0; j < V; j++)
#pragma unroll
                    for (int i = 0; i < E; i++) h[j].e[i] = dz_from_float<T>(dz_to_float(h[j].e[i]) + dz_to_float(r[j].e[i]));
            }
        }
        const long long here = row;
        row += step;
        if (a.sum) {
            T* out = static_cast<T*>(a.sum) + here * a.lds;
#pragma unroll
            for (int j = 0; j < V; j++) {
                if (WIDE) {
                    if (place(j, 0) < a.width) *reinterpret_cast<uint4*>(out + place(j, 0)) = h[j].q;
                } else {
#pragma unroll
                    for (int i = 0; i < E; i++)
                        if (place(j, i) < a.width) out[place(j, i)] = h[j].e[i];
                }
            }
        }
        float sum = 0.0f, top = 0.0f, u[V][E];
#pragma unroll
        for (int j = 0; j < V; j++) {
            float g[E];
            if (!KEPT) gains(j, g);
#pragma unroll
            for (int i = 0; i < E; i++) {
                const float v = dz_to_float(h[j].e[i]);
                sum = fmaf(v, v, sum);
                u[j][i] = __fmul_rn(KEPT ? kept[KEPT ? j : 0][i] : g[i], v);
                top = q8_larger(top, u[j][i]);
            }
        }
        q8_reduce<TEAM>(sum, top, turn);
        double mean = (double)sum;
        if (a.norm && q8_doubtful(sum)) {    // the whole team alike
            mean = 0.0;
#pragma unroll
            for (int j = 0; j < V; j++)
#pragma unroll
                for (int i = 0; i < E; i++) mean += (double)dz_to_float(h[j].e[i]) * (double)dz_to_float(h[j].e[i]);
            float same = top;
            q8_reduce<TEAM>(mean, same, turn);
        }
        const Q8Row k = q8_row(top);
        int8_t* codes = a.codes + here * a.ldc;
        auto write = [&](auto code) {
#pragma unroll
            for (int j = 0; j < V; j++) {
                if (place(j, 0) >= a.width) break;
                int c[E];
#pragma unroll
                for (int i = 0; i < E; i++) c[i] = code(u[j][i]);
                if (WIDE) {
                    unsigned word[E / 4];
#pragma unroll
                    for (int i = 0; i < E; i += 4)
                        word[i / 4] = __byte_perm(__byte_perm(c[i], c[i + 1], 0x0040), __byte_perm(c[i + 2], c[i + 3], 0x0040), 0x5410);
                    if (E == 8)
                        *reinterpret_cast<uint2*>(codes + place(j, 0)) = make_uint2(word[0], word[E / 4 - 1]);
                    else
                        *reinterpret_cast<unsigned*>(codes + place(j, 0)) = word[0];
                } else {
#pragma unroll
                    for (int i = 0; i < E; i++)
                        if (place(j, i) < a.width) codes[place(j, i)] = (int8_t)c[i];
                }
            }
        };
        if (k.plain)
            write([&](float v) { return q8_round(__fmul_rn(v, k.inverse)); });
        else
            write([&](float v) { return q8_code(k, v); });
        if (t == 0) a.scales[here] = q8_scale(a, top, mean / a.width);
        if (row >= a.rows) return;
    }
}

// Rows of any width, read again for their codes.
template <typename T> __global__ void __launch_bounds__(Q8N_THREADS) dz_norm_q8_long_kernel(const __grid_constant__ Q8NormArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.ldr : nullptr;
    T* out = a.sum ? static_cast<T*>(a.sum) + row * a.lds : nullptr;
    auto value = [&](int i) { return res ? dz_from_float<T>(dz_to_float(x[i]) + dz_to_float(res[i])) : x[i]; };
    double sum = 0.0;
    float top = 0.0f;
#pragma unroll 4
    for (int i = threadIdx.x; i < a.width; i += Q8N_THREADS) {
        const T h = value(i);
        const float v = dz_to_float(h);
        if (out) out[i] = h;                 // the same thread reads it below
        sum += (double)v * (double)v;
        top = q8_larger(top, a.gain ? __fmul_rn(a.gain[i], v) : v);
    }
    q8_reduce<Q8N_THREADS>(sum, top, 0);
    const Q8Row k = q8_row(top);
    int8_t* codes = a.codes + row * a.ldc;
#pragma unroll 4
    for (int i = threadIdx.x; i < a.width; i += Q8N_THREADS) {
        const float v = dz_to_float(out ? out[i] : value(i));
        codes[i] = (int8_t)q8_code(k, a.gain ? __fmul_rn(a.gain[i], v) : v);
    }
    if (threadIdx.x == 0) a.scales[row] = q8_scale(a, top, sum / a.width);
}

template <typename T, int TEAM, int V>
static cudaError_t q8_norm_v(const Q8NormArgs& a, bool wide, int device, int sms, cudaLaunchConfig_t& cfg) {
    static std::atomic<bool> ready[Q8N_DEVICES];
    if (wide && !ready[device].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(dz_norm_q8_kernel<T, TEAM, V, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   Q8Ring<V>::SMEM);
        if (e != cudaSuccess) return e;
        ready[device].store(true, std::memory_order_release);
    }
    // blocks that stay: as many as the SMs hold at once
    const long long each = Q8N_THREADS / TEAM, need = (a.rows + each - 1) / each, most = (long long)sms * Q8Ring<V>::BLOCKS;
    cfg.gridDim = dim3((unsigned)(need < most ? need : most));
    cfg.dynamicSmemBytes = wide ? Q8Ring<V>::SMEM : 0;
    return wide ? cudaLaunchKernelEx(&cfg, dz_norm_q8_kernel<T, TEAM, V, true>, a)
                : cudaLaunchKernelEx(&cfg, dz_norm_q8_kernel<T, TEAM, V, false>, a);
}

template <typename T> static cudaError_t q8_norm_t(const Q8NormArgs& a, bool wide, int device, int sms, cudaStream_t st) {
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
    if (vectors <= 32) return q8_norm_v<T, 32, 1>(a, wide, device, sms, cfg);
    if (vectors <= 64) return q8_norm_v<T, 32, 2>(a, wide, device, sms, cfg);
    if (vectors <= 256) return q8_norm_v<T, 256, 1>(a, wide, device, sms, cfg);
    if (vectors <= 512) return q8_norm_v<T, 256, 2>(a, wide, device, sms, cfg);
    if (vectors <= 1024) return q8_norm_v<T, 256, 4>(a, wide, device, sms, cfg);
    if (vectors <= 2048) return q8_norm_v<T, 256, 8>(a, wide, device, sms, cfg);
    cfg.gridDim = dim3((unsigned)a.rows);
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
    const bool wide = bases % 16 == 0 && (a.ldx | a.ldr | a.lds | (long long)width) * (long long)type_bytes(p->type) % 16 == 0 &&
                      ((uintptr_t)p->codes | (uintptr_t)a.ldc) % 8 == 0;
    if (p->device >= Q8N_DEVICES) return fail(DZ_E_UNSUPPORTED, "norm_q8: device ordinals below %d", Q8N_DEVICES);
    static std::atomic<int> known[Q8N_DEVICES];       // SM count per device, looked up once
    int sms = known[p->device].load(std::memory_order_relaxed);
    if (!sms) {
        DZ_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, p->device));
        known[p->device].store(sms, std::memory_order_relaxed);
    }
    cudaStream_t st = (cudaStream_t)stream;
    DZ_CUDA(p->type == DZ_TYPE_F32   ? q8_norm_t<float>(a, wide, p->device, sms, st)
            : p->type == DZ_TYPE_F16 ? q8_norm_t<__half>(a, wide, p->device, sms, st)
                                     : q8_norm_t<__nv_bfloat16>(a, wide, p->device, sms, st));
    return DZ_OK;
}
