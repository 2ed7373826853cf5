// The 4-bit ring caches' kernels (kv4.cuh) and C entry points, in a
// translation unit of their own.
#include "dz_cuda.h"

#include <cmath>

#include "kv4.cuh"
#include "shim.cuh"

namespace dz {

// ------------------------------------------------------------------- append

// One warp per (row, head), heads in the order queries, keys, values; lane l
// holds elements E l .. E l + E - 1 of the head (E = head_dim / 32). Queries
// are normed and rotated in fp32. Keys are in 64 bits up to one rounding to
// fp32, because the codes that follow round values next to a border and two
// summation orders would otherwise give different codes.
template <typename T, int E, typename A>
__device__ __forceinline__ void kv4_norm_rotate(A* x, const float* gain, const Kv4AppendArgs& a, long long pos,
                                                int lane) {
    constexpr int HD = 32 * E;
    if (gain) {
        A s = 0;
#pragma unroll
        for (int i = 0; i < E; i++) s += x[i] * x[i];
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        const A r = (A)1 / sqrt(s / (A)HD + (A)a.eps);
#pragma unroll
        for (int i = 0; i < E; i++) x[i] = (A)gain[lane * E + i] * x[i] * r;
    }
    if (!a.rope) return;
    if (a.halves) {
        // element e pairs with e + HD / 2, which lane + 16 holds at the same index
#pragma unroll
        for (int i = 0; i < E; i++) {
            double c, d;
            sincos((double)pos * a.freq[(lane & 15) * E + i], &d, &c);
            const A other = __shfl_xor_sync(0xffffffffu, x[i], 16);
            x[i] = lane < 16 ? x[i] * (A)c - other * (A)d : other * (A)d + x[i] * (A)c;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            double c, d;
            sincos((double)pos * a.freq[(lane * E + i) / 2], &d, &c);
            const A u = x[i], v = x[i + 1];
            x[i] = u * (A)c - v * (A)d;
            x[i + 1] = u * (A)d + v * (A)c;
        }
    }
}

// Quantizes a row of fp32 values and writes its codes and scales at `slot` of
// (b, h); x becomes the values that the codes stand for.
template <int E>
__device__ __forceinline__ void kv4_store_row(float* x, uint8_t* codes, float* scales, const Kv4Cache& c, int b, int h,
                                              long long slot, int lane) {
    constexpr int HD = 32 * E, LANES = KV4_GROUP / E;   // lanes of one group
    float peak = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < E; i++) {
        peak = fmaxf(peak, fabsf(x[i]));
        bad |= !(fabsf(x[i]) <= 3.402823466e38f);
    }
#pragma unroll
    for (int off = LANES / 2; off >= 1; off >>= 1) peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, off));
    const unsigned mask = LANES == 32 ? 0xffffffffu : (lane < 16 ? 0x0000ffffu : 0xffff0000u);
    const bool poisoned = __ballot_sync(0xffffffffu, bad) & mask;
    const float inverse = __fdiv_rn(7.0f, peak);
    const float scale = poisoned ? __int_as_float(0x7fc00000) : __fdiv_rn(peak, 7.0f);
    unsigned word = 0;
#pragma unroll
    for (int i = 0; i < E; i++) {
        const float v = __fmul_rn(x[i], inverse);
        float level = v >= 0.0f ? floorf(__fadd_rn(v, 0.5f)) : ceilf(__fsub_rn(v, 0.5f));
        level = fminf(fmaxf(level, -7.0f), 7.0f);
        if (poisoned || !(peak > 0.0f) || v != v) level = 0.0f;
        word |= (unsigned)((int)level + 7) << (4 * i);
        x[i] = level * scale;
    }
    const long long row = ((long long)b * c.kv_heads + h) * c.capacity + slot;
    if (E == 4)
        *reinterpret_cast<uint16_t*>(codes + row * (HD / 2) + 2 * lane) = (uint16_t)word;
    else
        codes[row * (HD / 2) + lane] = (uint8_t)word;
    if (lane % LANES == 0) scales[row * (HD / KV4_GROUP) + lane / LANES] = scale;
}

constexpr int KV4_APPEND_WARPS = 4;

template <typename T, int E>
__global__ void __launch_bounds__(KV4_APPEND_WARPS * 32) dz_kv4_append_kernel(const __grid_constant__ Kv4AppendArgs a) {
    constexpr int HD = 32 * E;
    const int lane = threadIdx.x & 31;
    const int heads = a.q_heads + 2 * a.c.kv_heads;
    const long long unit = (long long)blockIdx.x * KV4_APPEND_WARPS + (threadIdx.x >> 5);
    const long long row = unit / heads;
    int h = (int)(unit % heads);
    if (row >= (long long)a.c.batch * a.n_tokens) return;
    const int b = (int)(row / a.n_tokens), j = (int)(row % a.n_tokens);
    const long long first = a.positions[b];
    if (first < 0) return;
    const long long pos = first + j;
    const int kind = h < a.q_heads ? 0 : h < a.q_heads + a.c.kv_heads ? 1 : 2;
    h -= kind == 0 ? 0 : kind == 1 ? a.q_heads : a.q_heads + a.c.kv_heads;
    const T* in = static_cast<const T*>(kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                  row * (kind == 0 ? a.ldq : kind == 1 ? a.ldk : a.ldv) + (long long)h * HD + lane * E;
    T* out = static_cast<T*>(kind == 0 ? a.q_out : kind == 1 ? a.k_out : a.v_out);
    if (out) out += row * (kind == 0 ? a.ldqo : kind == 1 ? a.ldko : a.ldvo) + (long long)h * HD + lane * E;
    float x[E];
#pragma unroll
    for (int i = 0; i < E; i++) x[i] = dz_to_float(in[i]);
    if (kind == 0) {
        kv4_norm_rotate<T, E, float>(x, a.q_gain, a, pos, lane);
    } else {
        if (kind == 1) {
            double y[E];
#pragma unroll
            for (int i = 0; i < E; i++) y[i] = (double)x[i];
            kv4_norm_rotate<T, E, double>(y, a.k_gain, a, pos, lane);
#pragma unroll
            for (int i = 0; i < E; i++) x[i] = (float)y[i];
        }
        const long long slot = kv4_slot(pos, a.c.sinks, a.c.capacity - a.c.sinks);
        kv4_store_row<E>(x, kind == 1 ? a.c.k_codes : a.c.v_codes, kind == 1 ? a.c.k_scales : a.c.v_scales, a.c, b, h,
                         slot, lane);
    }
    if (out) {
#pragma unroll
        for (int i = 0; i < E; i++) out[i] = dz_from_float<T>(x[i]);
    }
}

template <typename T> static void kv4_append_t(const Kv4AppendArgs& a, int head_dim, unsigned grid, cudaStream_t st) {
    if (head_dim == 128)
        dz_kv4_append_kernel<T, 4><<<grid, KV4_APPEND_WARPS * 32, 0, st>>>(a);
    else
        dz_kv4_append_kernel<T, 2><<<grid, KV4_APPEND_WARPS * 32, 0, st>>>(a);
}

cudaError_t dz_kv4_append_launch(const Kv4AppendArgs& a, int type, int head_dim, cudaStream_t st) {
    const long long units = (long long)a.c.batch * a.n_tokens * (a.q_heads + 2 * a.c.kv_heads);
    const unsigned grid = (unsigned)((units + KV4_APPEND_WARPS - 1) / KV4_APPEND_WARPS);
    if (type == DZ_TYPE_F32)
        kv4_append_t<float>(a, head_dim, grid, st);
    else if (type == DZ_TYPE_F16)
        kv4_append_t<__half>(a, head_dim, grid, st);
    else
        kv4_append_t<__nv_bfloat16>(a, head_dim, grid, st);
    return cudaGetLastError();
}

}  // namespace dz

using namespace dz;

// The limits keep every index of a launch in range: rows x heads below 2^31
// warps, one cache buffer below 2^62 bytes.
static int kv4_check(const dz_kv4_t* c, const int64_t* positions, size_t n_tokens, Kv4Cache* out) {
    if (!c || !c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales || !positions)
        return fail(DZ_E_INVALID, "kv4: null argument");
    if (c->head_dim != 64 && c->head_dim != 128)
        return fail(DZ_E_UNSUPPORTED, "kv4: head dimension %zu (64 and 128 are supported)", c->head_dim);
    if (c->batch == 0 || c->batch > 65535 || c->kv_heads == 0 || c->kv_heads > 65535)
        return fail(DZ_E_INVALID, "kv4: batch and kv_heads must be 1..65535");
    if (c->capacity == 0 || c->capacity > INT32_MAX || c->sinks >= c->capacity)
        return fail(DZ_E_INVALID, "kv4: capacity must be 1..2^31-1 and sinks below it");
    if (n_tokens == 0 || n_tokens > c->capacity - c->sinks)
        return fail(DZ_E_INVALID, "kv4: n_tokens must be 1..capacity - sinks (%zu)", c->capacity - c->sinks);
    if ((((uintptr_t)c->k_codes | (uintptr_t)c->v_codes) & 15) || (((uintptr_t)c->k_scales | (uintptr_t)c->v_scales) & 7) ||
        ((uintptr_t)positions & 7))
        return fail(DZ_E_INVALID, "kv4: code buffers must be 16-byte aligned, scales and positions 8-byte aligned");
    *out = Kv4Cache{c->k_codes, c->v_codes, c->k_scales, c->v_scales, (int)c->batch, (int)c->kv_heads,
                    (long long)c->capacity, (long long)c->sinks};
    return DZ_OK;
}

// A typed row-strided operand: base aligned to its type, rows that hold their
// heads (or a single row), offsets in range.
static int kv4_rows(const char* what, const void* base, size_t stride, size_t heads, size_t head_dim, int type) {
    if (!base) return fail(DZ_E_INVALID, "kv4: %s is null", what);
    if ((uintptr_t)base % type_bytes(type)) return fail(DZ_E_INVALID, "kv4: %s is not aligned to its type", what);
    if (stride < heads * head_dim || stride > (1ull << 40))
        return fail(DZ_E_INVALID, "kv4: %s rows of %zu elements do not hold %zu heads", what, stride, heads);
    return DZ_OK;
}

extern "C" int dz_cuda_kv4_append(const dz_kv4_t* c, const dz_kv4_append_t* p, const int64_t* positions,
                                  size_t n_tokens, void* stream) {
    Kv4AppendArgs a;
    if (!p) return fail(DZ_E_INVALID, "kv4: null argument");
    int rc = kv4_check(c, positions, n_tokens, &a.c);
    if (rc) return rc;
    if (!type_ok(p->type)) return fail(DZ_E_INVALID, "kv4: unknown element type %d", p->type);
    if (p->q_heads > 65535 ||
        c->batch * n_tokens > (size_t)INT32_MAX / (p->q_heads + 2 * c->kv_heads))
        return fail(DZ_E_INVALID, "kv4: too many rows x heads in one call");
    if (p->q_heads) {
        if ((rc = kv4_rows("q", p->q, p->q_stride, p->q_heads, c->head_dim, p->type))) return rc;
        if ((rc = kv4_rows("q_out", p->q_out, p->q_out_stride, p->q_heads, c->head_dim, p->type))) return rc;
    }
    if ((rc = kv4_rows("k", p->k, p->k_stride, c->kv_heads, c->head_dim, p->type))) return rc;
    if ((rc = kv4_rows("v", p->v, p->v_stride, c->kv_heads, c->head_dim, p->type))) return rc;
    if (p->k_out && (rc = kv4_rows("k_out", p->k_out, p->k_out_stride, c->kv_heads, c->head_dim, p->type))) return rc;
    if (p->v_out && (rc = kv4_rows("v_out", p->v_out, p->v_out_stride, c->kv_heads, c->head_dim, p->type))) return rc;
    if ((p->q_gain || p->k_gain) && !(p->eps >= 0.0 && std::isfinite(p->eps)))
        return fail(DZ_E_INVALID, "kv4: the norm's eps must be finite and >= 0");
    if (((uintptr_t)p->q_gain | (uintptr_t)p->k_gain) & 3) return fail(DZ_E_INVALID, "kv4: gains are not aligned");
    if (p->rope_base != 0.0 && !(p->rope_base > 0.0 && std::isfinite(p->rope_base)))
        return fail(DZ_E_INVALID, "kv4: rope_base must be 0 (no rotation) or positive");
    if (p->rope_pairing != DZ_ROPE_PAIRS && p->rope_pairing != DZ_ROPE_HALVES)
        return fail(DZ_E_INVALID, "kv4: unknown rotation pairing %d", p->rope_pairing);
    DeviceGuard g(c->device);
    if (!g.ok) return fail(DZ_E_DEVICE, "cannot select device %d", c->device);
    a.positions = (const long long*)positions;
    a.q = p->q;
    a.k = p->k;
    a.v = p->v;
    a.q_out = p->q_out;
    a.k_out = p->k_out;
    a.v_out = p->v_out;
    a.ldq = (long long)p->q_stride;
    a.ldk = (long long)p->k_stride;
    a.ldv = (long long)p->v_stride;
    a.ldqo = (long long)p->q_out_stride;
    a.ldko = (long long)p->k_out_stride;
    a.ldvo = (long long)p->v_out_stride;
    a.q_gain = p->q_gain;
    a.k_gain = p->k_gain;
    a.eps = p->eps;
    a.n_tokens = (int)n_tokens;
    a.q_heads = (int)p->q_heads;
    a.rope = p->rope_base != 0.0;
    a.halves = p->rope_pairing == DZ_ROPE_HALVES;
    for (size_t i = 0; i < 64; i++)
        a.freq[i] = a.rope && i < c->head_dim / 2 ? pow(p->rope_base, -2.0 * (double)i / (double)c->head_dim) : 0.0;
    DZ_CUDA(dz_kv4_append_launch(a, p->type, (int)c->head_dim, (cudaStream_t)stream));
    return DZ_OK;
}

extern "C" int dz_cuda_kv4_attention(const dz_kv4_t* c, const dz_kv4_attention_t* p, const int64_t* positions,
                                     size_t n_tokens, void* stream) {
    Kv4AttnArgs a;
    if (!p) return fail(DZ_E_INVALID, "kv4: null argument");
    int rc = kv4_check(c, positions, n_tokens, &a.c);
    if (rc) return rc;
    if (!type_ok(p->type)) return fail(DZ_E_INVALID, "kv4: unknown element type %d", p->type);
    if (p->q_heads == 0 || p->q_heads > 65535 || p->q_heads % c->kv_heads)
        return fail(DZ_E_INVALID, "kv4: q_heads must be a multiple of kv_heads");
    if (c->batch * n_tokens > (size_t)INT32_MAX / p->q_heads)
        return fail(DZ_E_INVALID, "kv4: too many rows x heads in one call");
    if ((rc = kv4_rows("q", p->q, p->q_stride, p->q_heads, c->head_dim, p->type))) return rc;
    if ((rc = kv4_rows("out", p->out, p->out_stride, p->q_heads, c->head_dim, p->type))) return rc;
    if (!std::isfinite(p->scale)) return fail(DZ_E_INVALID, "kv4: scale must be finite");
    if (p->window && (p->window > c->capacity - c->sinks || p->window + n_tokens - 1 > c->capacity - c->sinks))
        return fail(DZ_E_INVALID, "kv4: window + n_tokens - 1 must be at most capacity - sinks (%zu)",
                    c->capacity - c->sinks);
    DeviceGuard g(c->device);
    if (!g.ok) return fail(DZ_E_DEVICE, "cannot select device %d", c->device);
    a.positions = (const long long*)positions;
    a.q = p->q;
    a.out = p->out;
    a.ldq = (long long)p->q_stride;
    a.ldo = (long long)p->out_stride;
    a.n_tokens = (int)n_tokens;
    a.q_heads = (int)p->q_heads;
    a.scale = p->scale;
    a.window = (long long)p->window;
    DZ_CUDA(dz_kv4_attn_launch(a, p->type, (int)c->head_dim, c->device, (cudaStream_t)stream));
    return DZ_OK;
}
