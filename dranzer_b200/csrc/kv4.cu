// The 4-bit ring caches' kernels (kv4.cuh) and C entry points, in a
// translation unit of their own.
#include "dz_cuda.h"

#include <atomic>
#include <cmath>
#include <cstring>

#include "headrows.cuh"
#include "kv4.cuh"
#include "shim.cuh"

namespace dz {

// ------------------------------------------------------------------- append
//
// A block of eight warps takes up to 256 / (head_dim / 2) rows (tokens of
// sequences), or a share of one row's heads, in the order queries, keys,
// values; the rows' angles are computed once, a thread per pair, and shared. A
// lane holds 16 bytes of a head, so a warp takes 1, 2 or 4 heads at a time and
// loads the next ones while it works. Bound by HBM for many rows and by
// latency for few: rows and their heads spread over more blocks until the SMs
// are full. 7600 rows of 48 heads of 64 (bf16): 38 us, against 15 us of bytes;
// sine and cosine in 64 bits for each warp and head again took 152 us, a row to
// a block 77 us, the kinds of heads mixed in one loop 47 us. What is left is
// instructions (28 M at 2.5 a cycle); loads two items ahead changed nothing.
//
// Queries are normed and rotated in fp32. Keys are in 64 bits up to one
// rounding to fp32, because the codes that follow round values next to a
// border and two summation orders would otherwise give different codes.

constexpr int KV4_APPEND_WARPS = 8;

// Where the angle of pair p lies in a row's table: the pairs of one lane that
// its i-th step turns lie side by side over the lanes.
template <int HD, int E> __device__ __forceinline__ int kv4_angle_at(int p, bool halves) {
    const int own = halves ? E : E / 2;      // pairs of a lane
    return p % own * (HD / 2 / own) + p / own;
}

__device__ __forceinline__ float kv4_signed(float v, bool minus) {
    return __uint_as_float(__float_as_uint(v) ^ (minus ? 0x80000000u : 0u));
}
__device__ __forceinline__ double kv4_signed(double v, bool minus) {
    return __hiloint2double(__double2hiint(v) ^ (minus ? (int)0x80000000 : 0), __double2loint(v));
}

// Rotates a head's E elements of this lane, element `at` first; angle(i) gives
// cosine and sine of the lane's i-th pair.
template <int HD, int E, typename A, typename F>
__device__ __forceinline__ void kv4_rotate(A (&x)[E], bool halves, int lane, int at, F angle) {
    constexpr int LPH = HD / E;
    if (halves) {
        // element e pairs with e + HD / 2, which the lane half a head away holds at the same index:
        // x cos - other sin in the first half, x cos + other sin in the second
        const unsigned mask = kv4_mask<LPH>(lane);
#pragma unroll
        for (int i = 0; i < E; i++) {
            const auto q = angle(i);
            const A other = kv4_signed(__shfl_xor_sync(mask, x[i], LPH / 2), at < HD / 2);
            x[i] = x[i] * (A)q.x + other * (A)q.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            const auto q = angle(i / 2);
            const A u = x[i], v = x[i + 1];
            x[i] = u * (A)q.x - v * (A)q.y;
            x[i + 1] = u * (A)q.y + v * (A)q.x;
        }
    }
}

// Quantizes the lane's elements of a row and writes their codes (and the
// group's scale) at cache row `row`; x becomes the values that they stand for.
template <int HD, int E>
__device__ __forceinline__ void kv4_store_row(float (&x)[E], uint8_t* codes, float* scales, long long row, int lane,
                                              int at) {
    constexpr int LANES = KV4_GROUP / E;     // lanes of a group
    const unsigned mask = kv4_mask<LANES>(lane);
    unsigned top = 0;                        // bits of the largest magnitude; above 0x7f7fffff it is not finite
#pragma unroll
    for (int i = 0; i < E; i++) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
    for (int off = LANES / 2; off >= 1; off >>= 1) top = max(top, __shfl_xor_sync(mask, top, off));
    const bool poisoned = top > 0x7f7fffffu;
    const float peak = __uint_as_float(top), inverse = __fdiv_rn(7.0f, peak);
    const float scale = poisoned ? __int_as_float(0x7fc00000) : __fdiv_rn(peak, 7.0f);
    unsigned word = 0;
    if (poisoned || !(inverse <= 3.402823466e38f)) {
        // not finite, all zero, or a peak below 2e-38 (whose inverse overflows: zeros give NaN, level 0, the rest +-7)
#pragma unroll
        for (int i = 0; i < E; i++) {
            const float v = __fmul_rn(x[i], inverse);
            const float level = poisoned || top == 0 || v != v ? 0.0f : copysignf(7.0f, v);
            word |= (unsigned)((int)level + 7) << (4 * i);
            x[i] = level * scale;
        }
    } else {
        // |x| <= peak, so the scaled value is at most 7 and two roundings, and needs no clamp
#pragma unroll
        for (int i = 0; i < E; i++) {
            const float v = __fmul_rn(x[i], inverse);
            const unsigned code = (unsigned)(__float2int_rz(__fadd_rn(v, copysignf(0.5f, v))) + 7);   // half away from zero
            word += code << (4 * i);
            x[i] = (__uint_as_float(0x4B000000u | code) - 8388615.0f) * scale;   // 2^23 + code, less 2^23 + 7
        }
    }
    uint8_t* to = codes + row * (HD / 2) + at / 2;
    if (E == 8)
        *reinterpret_cast<uint32_t*>(to) = word;
    else
        *reinterpret_cast<uint16_t*>(to) = (uint16_t)word;
    if (at % KV4_GROUP == 0) scales[row * (HD / KV4_GROUP) + at / KV4_GROUP] = scale;
}

// How a launch is cut: blocks take `rows` rows each (a power of two), or
// `parts` blocks share one row.
struct Kv4AppendCut {
    int rows, parts;
    int wide;                   // every row of every operand starts on a 16-byte boundary
};

template <typename T, int HD>
__global__ void __launch_bounds__(KV4_APPEND_WARPS * 32, 3) dz_kv4_append_kernel(const __grid_constant__ Kv4AppendArgs a,
                                                                                const __grid_constant__ Kv4AppendCut cut) {
    constexpr int E = 16 / (int)sizeof(T), LPH = HD / E, HPW = 32 / LPH;   // elements, lanes of a head, heads of a warp
    constexpr int THREADS = KV4_APPEND_WARPS * 32, ROWS = THREADS / (HD / 2);
    asm volatile("griddepcontrol.wait;" ::: "memory");   // launched while the kernel before ends
    __shared__ double2 angles[ROWS][HD / 2];
    __shared__ float2 angles_f[ROWS][HD / 2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, at = lane % LPH * E, mine = lane / LPH;
    const int all_rows = a.c.batch * a.n_tokens;
    const int row0 = blockIdx.x / (unsigned)cut.parts * cut.rows, part = blockIdx.x % (unsigned)cut.parts;
    // the warp's row, and its items: a warp's worth of query heads, then of key heads, then of value heads each
    const int team = KV4_APPEND_WARPS / cut.rows, r = warp / team, row = row0 + r;
    const int nq = (a.q_heads + HPW - 1) / HPW, nk = (a.c.kv_heads + HPW - 1) / HPW;
    const int step = cut.parts * team;
    int item = part * team + warp % team;
    union Lane {                // 16 bytes of a head
        uint4 q;
        T e[E];
        __device__ Lane() {}
    };
    const T* qi = static_cast<const T*>(a.q) + row * a.ldq + mine * HD + at;
    const T* ki = static_cast<const T*>(a.k) + row * a.ldk + mine * HD + at;
    const T* vi = static_cast<const T*>(a.v) + row * a.ldv + mine * HD + at;
    auto load = [&](const T* in, Lane& io) {
        if (cut.wide) {
            io.q = *reinterpret_cast<const uint4*>(in);
        } else {
#pragma unroll
            for (int k = 0; k < E; k++) io.e[k] = in[k];
        }
    };
    auto fetch = [&](int i, Lane& io) {
        if (row >= all_rows) return;
        if (i < nq) {
            if (i * HPW + mine < a.q_heads) load(qi + i * (HPW * HD), io);
        } else if (i < nq + nk) {
            if ((i - nq) * HPW + mine < a.c.kv_heads) load(ki + (i - nq) * (HPW * HD), io);
        } else if ((i - nq - nk) * HPW + mine < a.c.kv_heads) {
            load(vi + (i - nq - nk) * (HPW * HD), io);
        }
    };
    auto store = [&](T* out, const float (&x)[E]) {
        Lane io;
#pragma unroll
        for (int i = 0; i < E; i++) io.e[i] = dz_from_float<T>(x[i]);
        if (cut.wide) {
            *reinterpret_cast<uint4*>(out) = io.q;
        } else {
#pragma unroll
            for (int i = 0; i < E; i++) out[i] = io.e[i];
        }
    };
    Lane io, next;
    fetch(item, next);
    if (a.rope) {
        for (int i = threadIdx.x; i < cut.rows * (HD / 2); i += THREADS) {
            const int rr = i / (HD / 2), p = i % (HD / 2), w = min(row0 + rr, all_rows - 1);
            double c, s;
            sincos((double)(a.positions[w / a.n_tokens] + a.pos_add + w % a.n_tokens) * a.freq[p], &s, &c);
            const int to = kv4_angle_at<HD, E>(p, a.halves);
            angles[rr][to] = make_double2(c, s);
            angles_f[rr][to] = make_float2((float)c, (float)s);
        }
        __syncthreads();
    }
    if (row >= all_rows) return;
    const int b = row / a.n_tokens;
    const long long first = a.positions[b] + a.pos_add;
    if (kv4_skips(first)) return;
    // the lane's place in the angle table
    const int stride = a.halves ? HD / 2 / E : LPH, place = a.halves ? at % (HD / 2) / E : at / E;

    if (item < nq) {
        float2 turn[E];         // E / 2 of them when pairs lie side by side
        float gain[E];
#pragma unroll
        for (int i = 0; i < E; i++) {
            if (a.rope && (a.halves || i < E / 2)) turn[i] = angles_f[r][i * stride + place];
            gain[i] = a.q_gain ? a.q_gain[at + i] : 1.0f;
        }
        T* out = static_cast<T*>(a.q_out) + row * a.ldqo + at;
        for (; item < nq; item += step) {
            io.q = next.q;
            fetch(item + step, next);
            const int h = item * HPW + mine;
            if (h >= a.q_heads) continue;   // whole heads: a head's lanes stay together below
            float x[E];
#pragma unroll
            for (int i = 0; i < E; i++) x[i] = dz_to_float(io.e[i]);
            if (a.q_gain) {
                const unsigned mask = kv4_mask<LPH>(lane);
                const float s = kv4_square_sum<LPH>(x, mask);
                float n = kv4_rsqrt(s * (1.0f / HD) + (float)a.eps);
                if (!(s > 1e-25f && s < 1e37f)) {   // squares that leave fp32's range
                    double y[E];
#pragma unroll
                    for (int i = 0; i < E; i++) y[i] = (double)x[i];
                    const double m = kv4_square_sum<LPH>(y, mask) / HD + a.eps;
#pragma unroll
                    for (int i = 0; i < E; i++) x[i] = (float)(y[i] * kv4_rsqrt(m));
                    n = 1.0f;
                }
#pragma unroll
                for (int i = 0; i < E; i++) x[i] = gain[i] * (x[i] * n);   // x n is about 1: gains of any size
            }
            if (a.rope) kv4_rotate<HD>(x, a.halves, lane, at, [&](int i) { return turn[i]; });
            store(out + h * HD, x);
        }
    }
    const long long pos = first + (row - b * a.n_tokens);
    // the row's place in key head 0 of the cache
    const long long place0 = (long long)b * a.c.kv_heads * a.c.capacity + kv4_slot(pos, a.c.sinks, a.c.capacity - a.c.sinks);
    for (; item < nq + nk; item += step) {
        io.q = next.q;
        fetch(item + step, next);
        const int h = (item - nq) * HPW + mine;
        if (h >= a.c.kv_heads) continue;
        double y[E];
#pragma unroll
        for (int i = 0; i < E; i++) y[i] = (double)dz_to_float(io.e[i]);
        if (a.k_gain) {
            const double n = kv4_rsqrt(kv4_square_sum<LPH>(y, kv4_mask<LPH>(lane)) / HD + a.eps);
#pragma unroll
            for (int i = 0; i < E; i++) y[i] = (double)a.k_gain[at + i] * y[i] * n;
        }
        if (a.rope) kv4_rotate<HD>(y, a.halves, lane, at, [&](int i) { return angles[r][i * stride + place]; });
        float x[E];
#pragma unroll
        for (int i = 0; i < E; i++) x[i] = (float)y[i];
        kv4_store_row<HD>(x, a.c.k_codes, a.c.k_scales, place0 + h * a.c.capacity, lane, at);
        if (a.k_out) store(static_cast<T*>(a.k_out) + row * a.ldko + h * HD + at, x);
    }
    for (; item < nq + 2 * nk; item += step) {
        io.q = next.q;
        fetch(item + step, next);
        const int h = (item - nq - nk) * HPW + mine;
        if (h >= a.c.kv_heads) continue;
        float x[E];
#pragma unroll
        for (int i = 0; i < E; i++) x[i] = dz_to_float(io.e[i]);
        kv4_store_row<HD>(x, a.c.v_codes, a.c.v_scales, place0 + h * a.c.capacity, lane, at);
        if (a.v_out) store(static_cast<T*>(a.v_out) + row * a.ldvo + h * HD + at, x);
    }
}

template <typename T, int HD> static cudaError_t kv4_append_t(const Kv4AppendArgs& a, int sms, cudaStream_t st) {
    constexpr int HPW = 32 * 16 / (int)sizeof(T) / HD, ROWS = KV4_APPEND_WARPS * 32 / (HD / 2);
    const long long rows = (long long)a.c.batch * a.n_tokens;
    const int groups = (a.q_heads + HPW - 1) / HPW + 2 * ((a.c.kv_heads + HPW - 1) / HPW);   // items of a row
    // eight blocks to an SM (several times what it holds) first, then more rows to a block
    Kv4AppendCut cut;
    const long long blocks = 8LL * sms, most = (groups + KV4_APPEND_WARPS - 1) / KV4_APPEND_WARPS;
    for (cut.rows = 1; cut.rows < ROWS && cut.rows < KV4_APPEND_WARPS && rows / (2 * cut.rows) >= blocks;) cut.rows *= 2;
    cut.parts = (int)(rows >= blocks ? 1 : (blocks + rows - 1) / rows > most ? most : (blocks + rows - 1) / rows);
    const uintptr_t bases = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.k_out |
                            (uintptr_t)a.v_out;
    const long long strides = a.ldq | a.ldk | a.ldv | a.ldqo | a.ldko | a.ldvo;
    cut.wide = bases % 16 == 0 && strides * (long long)sizeof(T) % 16 == 0;
    const unsigned grid = (unsigned)((rows + cut.rows - 1) / cut.rows * cut.parts);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(KV4_APPEND_WARPS * 32);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, dz_kv4_append_kernel<T, HD>, a, cut);
}

template <typename T> static cudaError_t kv4_append_h(const Kv4AppendArgs& a, int head_dim, int sms, cudaStream_t st) {
    return head_dim == 128 ? kv4_append_t<T, 128>(a, sms, st) : kv4_append_t<T, 64>(a, sms, st);
}

cudaError_t dz_kv4_append_launch(const Kv4AppendArgs& a, int type, int head_dim, int device, cudaStream_t st) {
    static std::atomic<int> known[64];       // SM count per device, looked up once
    int sms = device >= 0 && device < 64 ? known[device].load(std::memory_order_relaxed) : 0;
    if (!sms) {
        const cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
        if (e != cudaSuccess) return e;
        if (device >= 0 && device < 64) known[device].store(sms, std::memory_order_relaxed);
    }
    if (type == DZ_TYPE_F32) return kv4_append_h<float>(a, head_dim, sms, st);
    if (type == DZ_TYPE_F16) return kv4_append_h<__half>(a, head_dim, sms, st);
    return kv4_append_h<__nv_bfloat16>(a, head_dim, sms, st);
}

void dz_kv4_frequencies(double base, size_t head_dim, double* freq) {
    // the last ones are kept: 64 powers cost as much as a launch
    static thread_local struct { double base, freq[64]; size_t head_dim; } last = {-1.0, {}, 0};
    if (last.base != base || last.head_dim != head_dim) {
        for (size_t i = 0; i < 64; i++)
            last.freq[i] = base != 0.0 && i < head_dim / 2 ? pow(base, -2.0 * (double)i / (double)head_dim) : 0.0;
        last.base = base;
        last.head_dim = head_dim;
    }
    memcpy(freq, last.freq, sizeof(last.freq));
}

}  // namespace dz

using namespace dz;

// The limits keep every index of a launch in range: rows x heads below 2^31
// warps, one cache buffer of at most 2^62 bytes.
static int kv4_check(const dz_kv4_t* c, const int64_t* positions, size_t n_tokens, Kv4Cache* out) {
    if (!c || !c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales || !positions)
        return fail(DZ_E_INVALID, "kv4: null argument");
    if (c->head_dim != 64 && c->head_dim != 128)
        return fail(DZ_E_UNSUPPORTED, "kv4: head dimension %zu (64 and 128 are supported)", c->head_dim);
    if (c->batch == 0 || c->batch > 65535 || c->kv_heads == 0 || c->kv_heads > 65535)
        return fail(DZ_E_INVALID, "kv4: batch and kv_heads must be 1..65535");
    if (c->capacity == 0 || c->capacity > (size_t)KV4_CAPACITY || c->sinks >= c->capacity)
        return fail(DZ_E_INVALID, "kv4: capacity must be 1..2^31-64 and sinks below it");
    if (c->capacity > ((size_t)1 << 62) / (c->batch * c->kv_heads * (c->head_dim / 2)))
        return fail(DZ_E_INVALID, "kv4: a buffer of %zu x %zu rings of %zu rows is above 2^62 bytes", c->batch, c->kv_heads,
                    c->capacity);
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
// heads, offsets in range.
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
    a.pos_add = 0;
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
    dz_kv4_frequencies(p->rope_base, c->head_dim, a.freq);
    DZ_CUDA(dz_kv4_append_launch(a, p->type, (int)c->head_dim, c->device, (cudaStream_t)stream));
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
    a.pos_add = 0;
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
