// Attention over the 4-bit ring caches (kv4.cuh), in a translation unit of its
// own.
//
// One cluster of 1 to 8 blocks handles one (sequence, key head) and up to NT x
// 8 / PARTS of its (query token, query head) pairs; the visible tokens go in
// tiles of 32 to the cluster's warps in turn, each warp keeps its own softmax
// state, and the states join in shared memory, then across the cluster.
//
// Products. Codes become levels -7..7 in fp16, which is exact, in the A
// operand of mma.m16n8k16; the B columns are the pairs:
//   scores   A = 16 tokens x 16 elements of K, B = the query, per 64-element
//            group, each group's sum times the token's scale in fp32;
//   values   A = 16 elements of V^T x 16 tokens, B = weight x value scale.
// fp32 and fp16 queries and weights enter as two fp16 columns (PARTS = 2), hi
// = fp16(x) and lo = fp16(x - hi): 22 to 24 bits, so that products keep fp32
// accuracy; the query scaled by a power of two that puts its largest element
// in [2^14, 2^15). bf16 queries are exact in one column, and their weights are
// rounded to fp16's 11 bits (2^-12 relative, an eighth of the output's own
// rounding).
//
// Weights. p = 2^(x - m) against the pair's running maximum m; what enters the
// product is p x scale / R x 2^14, with R at least the largest p x scale of
// the pair so far (in units of 2^m). R follows the products themselves, not the
// scales alone, because a token that takes all the weight may hold nothing,
// as first tokens often do, and the rest then decides the result.
#include <atomic>
#include <cmath>

#include "kv4.cuh"
#include "shim.cuh"

namespace dz {

constexpr int KA_WARPS = 8;
constexpr int KA_TILE = 32;     // tokens of a tile
constexpr int KA_STAGES = 3;
constexpr float KA_TOP = 16384.0f;     // 2^14
constexpr int KA_DEVICES = 64;  // devices whose launch state is kept
constexpr float KA_RMIN = 1e-30f;

template <int HD> struct KaCfg {
    static constexpr int ROW = HD / 2;                 // code bytes of a row
    static constexpr int GROUPS = HD / KV4_GROUP;
    static constexpr int CODES = KA_TILE * ROW;
    static constexpr int SCALES = KA_TILE * GROUPS * 4;
    static constexpr int STAGE = 2 * CODES + 2 * SCALES;
    static constexpr int RING = KA_WARPS * KA_STAGES * STAGE;
};

__device__ __forceinline__ void ka_copy16(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? 16 : 0;   // 0: the 16 bytes are zeroed
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n));
}
template <int BYTES> __device__ __forceinline__ void ka_copy_small(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? BYTES : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n));
}
__device__ __forceinline__ void ka_commit() { asm volatile("cp.async.commit_group;"); }
template <int N> __device__ __forceinline__ void ka_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N)); }

__device__ __forceinline__ void ka_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ka_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Levels of the nibbles at bits 0 and 16 (low) or 4 and 20 (high) of w, as
// fp16 pairs. 0x6400 is 1024, whose step is 1: or-ing a nibble in adds it (or
// 16 x it), and the subtraction is exact.
__device__ __forceinline__ uint32_t ka_low(uint32_t w) {
    const uint32_t x = (w & 0x000F000Fu) | 0x64006400u;
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6407)));  // 1031
    return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ uint32_t ka_high(uint32_t w) {
    const uint32_t x = (w & 0x00F000F0u) | 0x64006400u;
    const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x2C00)),   // 1/16
                              __half2half2(__ushort_as_half(0xD470)));                                         // -71
    return *reinterpret_cast<const uint32_t*>(&y);
}

__device__ __forceinline__ uint32_t ka_pack(float a, float b) {   // a in the low half
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 ka_unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

// Column `part` of two values: hi, or what hi leaves.
template <int PARTS> __device__ __forceinline__ uint32_t ka_column(float a, float b, bool low) {
    const uint32_t hi = ka_pack(a, b);
    if (PARTS == 1) return hi;
    const float2 f = ka_unpack(hi);
    const uint32_t lo = ka_pack(a - f.x, b - f.y);
    return low ? lo : hi;
}

template <typename T, int HD, int PARTS, int NT>
__global__ void __launch_bounds__(KA_WARPS * 32, NT == 1 ? 2 : 1) dz_kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a,
                                                                                    int cluster, int pair_blocks) {
    using C = KaCfg<HD>;
    constexpr int NP = 2 / PARTS;            // pairs of a lane in one n-tile
    constexpr int PAIRS = NT * 8 / PARTS;    // pairs of a block
    constexpr int GR = C::GROUPS;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % cluster;
    int unit = blockIdx.x / cluster;
    const int pb = unit % pair_blocks;
    unit /= pair_blocks;
    const int hk = unit % a.c.kv_heads, b = unit / a.c.kv_heads;
    const long long first = a.positions[b];
    if (first < 0) return;                   // the whole cluster leaves
    const int share = a.q_heads / a.c.kv_heads, pairs = share * a.n_tokens, pair0 = pb * PAIRS;

    // ---- the virtual index v = 0..count-1 runs over the sinks, then over positions lo, lo + 1, ...
    const long long ring = a.c.capacity - a.c.sinks, last = first + a.n_tokens - 1;
    const int j_lo = pair0 / share, j_hi = min((pair0 + PAIRS - 1) / share, a.n_tokens - 1);
    const long long q_hi = first + j_hi;
    long long lo = max(a.c.sinks, last - ring + 1);
    if (a.window) lo = max(lo, first + j_lo - a.window + 1);
    const int nsink = (int)min(a.c.sinks, q_hi + 1);
    const int count = nsink + (int)max(0LL, q_hi + 1 - lo);
    const int start = (int)kv4_slot(lo, a.c.sinks, ring);     // slot of lo; the ring wraps at capacity
    const int cap = (int)a.c.capacity, iring = (int)ring;
    const long long base = ((long long)b * a.c.kv_heads + hk) * a.c.capacity;
    const uint8_t* kc = a.c.k_codes + base * C::ROW;
    const uint8_t* vc = a.c.v_codes + base * C::ROW;
    const float* ksc = a.c.k_scales + base * GR;
    const float* vsc = a.c.v_scales + base * GR;

    uint8_t* my = smem + warp * KA_STAGES * C::STAGE;
    const uint32_t my_s = (uint32_t)__cvta_generic_to_shared(my);
    auto slot_of = [&](int v) {
        if (v < nsink) return v;
        const unsigned s = (unsigned)(v - nsink) + (unsigned)start;   // both below 2^31
        return (int)(s >= (unsigned)cap ? s - (unsigned)iring : s);
    };
    // A tile's copies. Chunk c of row r lies at chunk c ^ (r & 2) (HD 128), so
    // that the fragment reads of K (8 rows x 32 bytes) and V (4 rows x 32
    // bytes) meet all banks once. Rows past `count` become zeros.
    constexpr int CH = C::ROW / 16, RPI = 32 / CH;            // chunks of a row, rows of one pass over the lanes
    auto issue = [&](int tile, int stage) {
        const uint32_t s = my_s + stage * C::STAGE;
        const int v0 = tile * KA_TILE;
#pragma unroll
        for (int i = 0; i < KA_TILE / RPI; i++) {
            const int r = lane / CH + i * RPI, c = lane % CH;
            const bool valid = v0 + r < count;
            const long long off = (long long)(valid ? slot_of(v0 + r) : 0) * C::ROW + c * 16;
            const uint32_t d = s + r * C::ROW + (HD == 128 ? (c ^ (r & 2)) : c) * 16;
            ka_copy16(d, kc + off, valid);
            ka_copy16(d + C::CODES, vc + off, valid);
        }
        const bool valid = v0 + lane < count;
        const long long off = (long long)(valid ? slot_of(v0 + lane) : 0) * GR;
        ka_copy_small<GR * 4>(s + 2 * C::CODES + lane * GR * 4, ksc + off, valid);
        ka_copy_small<GR * 4>(s + 2 * C::CODES + C::SCALES + lane * GR * 4, vsc + off, valid);
    };

    const int ntiles = (count + KA_TILE - 1) / KA_TILE, step = KA_WARPS * cluster;
    const int tile0 = rank * KA_WARPS + warp;
#pragma unroll
    for (int i = 0; i < KA_STAGES - 1; i++) {
        if (tile0 + i * step < ntiles) issue(tile0 + i * step, i);
        ka_commit();
    }

    // ---- query fragments: column g of n-tile n is part (g % PARTS) of pair
    // pair0 + n * 8 / PARTS + g / PARTS; the lane's elements follow the order in
    // which a code word's nibbles become A registers
    uint32_t qf[NT][GR * 4][2];
    float qfac[NT];                          // scale x log2 e / the pair's power of two, column layout (g)
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int pair = pair0 + n * (8 / PARTS) + g / PARTS;
        const bool live = pair < pairs;
        const T* q = static_cast<const T*>(a.q) +
                     ((long long)b * a.n_tokens + (live ? pair / share : 0)) * a.ldq +
                     (long long)(hk * share + (live ? pair % share : 0)) * HD;
        float x[GR * 16];
        float top = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < GR * 16; i++) {
            x[i] = live ? dz_to_float(q[(i / 16) * 64 + 16 * t + i % 16]) : 0.0f;
            top = fmaxf(top, fabsf(x[i]));
            bad |= !(fabsf(x[i]) <= 3.402823466e38f);
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        bad = __any_sync(0xfu << (lane & 28), bad);
        // 2^(14 - e) for top in [2^e, 2^(e+1)), as a product of two powers so that neither over- nor underflows
        int e = top > 0.0f && !bad ? ilogbf(top) : 0;
        e = max(e, -140);
        const int up = 14 - e, u0 = up / 2, u1 = up - u0;
        const float f0 = __int_as_float((127 + u0) << 23), f1 = __int_as_float((127 + u1) << 23);
        const float d0 = __int_as_float((127 - u0) << 23), d1 = __int_as_float((127 - u1) << 23);
        qfac[n] = bad ? __int_as_float(0x7fc00000) : a.scale * 1.4426950408889634f * d0 * d1;
#pragma unroll
        for (int w = 0; w < GR * 2; w++) {   // word w of the lane: elements 8 w .. 8 w + 7 of its x
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = x[8 * w + i] * f0 * f1;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                qf[n][2 * w + h][0] = ka_column<PARTS>(y[2 * h], y[2 * h + 4], g & 1);
                qf[n][2 * w + h][1] = ka_column<PARTS>(y[2 * h + 1], y[2 * h + 5], g & 1);
            }
        }
    }
    // ---- the same factor, and the visible range, of the lane's pairs in score layout (t)
    float sfac[NT][NP];
    int see_sink[NT][NP], see_hi[NT][NP], see_lo[NT][NP];
    const bool masked = a.n_tokens > 1;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int col = PARTS == 2 ? 2 * t : 2 * t + i;
            sfac[n][i] = __shfl_sync(0xffffffffu, qfac[n], col * 4);
            const int pair = min(pair0 + n * (8 / PARTS) + col / PARTS, pairs - 1);
            const long long pos = first + pair / share;
            see_sink[n][i] = (int)min(pos, (long long)INT32_MAX);
            see_hi[n][i] = (int)max(-1LL, pos - lo);
            see_lo[n][i] = a.window ? (int)max(-1LL, pos - a.window - lo) : -1;
        }

    float m[NT][NP], l[NT][NP], R[NT], rinv[NT];
    float acc[NT][GR * 4][4];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        R[n] = KA_RMIN;
        rinv[n] = KA_TOP / KA_RMIN;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            m[n][i] = -INFINITY;
            l[n][i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < GR * 4; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) acc[n][i][r] = 0.0f;
    }

    int stage = 0, next = KA_STAGES - 1;
    for (int tile = tile0; tile < ntiles; tile += step) {
        ka_wait<KA_STAGES - 2>();
        __syncwarp();
        if (tile + (KA_STAGES - 1) * step < ntiles) issue(tile + (KA_STAGES - 1) * step, next);
        ka_commit();
        const uint8_t* st = my + stage * C::STAGE;
        stage = stage + 1 == KA_STAGES ? 0 : stage + 1;
        next = next + 1 == KA_STAGES ? 0 : next + 1;
        const float* ks = reinterpret_cast<const float*>(st + 2 * C::CODES);
        const float* vs = ks + KA_TILE * GR;

        // scores: x[n][blk][row half][pair]
        float x[NT][2][2][NP];
#pragma unroll
        for (int blk = 0; blk < 2; blk++) {
            const int r0 = blk * 16 + g, r1 = r0 + 8;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < NP; i++) x[n][blk][0][i] = x[n][blk][1][i] = 0.0f;
#pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                // 8 bytes at 8 t of the group's 32: rows r0 and r1 (r1 & 2 == r0 & 2)
                const int at = HD == 128 ? ((2 * gr + (t >> 1)) ^ (r0 & 2)) * 16 + 8 * (t & 1) : 8 * t;
                const uint2 w0 = *reinterpret_cast<const uint2*>(st + r0 * C::ROW + at);
                const uint2 w1 = *reinterpret_cast<const uint2*>(st + r1 * C::ROW + at);
                float s[NT][4];
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int r = 0; r < 4; r++) s[n][r] = 0.0f;
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const uint32_t p = u ? w0.y : w0.x, q = u ? w1.y : w1.x;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t a0 = ka_low(p >> (8 * h)), a2 = ka_high(p >> (8 * h));
                        const uint32_t a1 = ka_low(q >> (8 * h)), a3 = ka_high(q >> (8 * h));
#pragma unroll
                        for (int n = 0; n < NT; n++)
                            ka_mma(s[n], a0, a1, a2, a3, qf[n][4 * gr + 2 * u + h][0], qf[n][4 * gr + 2 * u + h][1]);
                    }
                }
                const float k0 = ks[r0 * GR + gr], k1 = ks[r1 * GR + gr];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    if (PARTS == 2) {
                        x[n][blk][0][0] = fmaf(s[n][0] + s[n][1], k0, x[n][blk][0][0]);
                        x[n][blk][1][0] = fmaf(s[n][2] + s[n][3], k1, x[n][blk][1][0]);
                    } else {
                        x[n][blk][0][0] = fmaf(s[n][0], k0, x[n][blk][0][0]);
                        x[n][blk][0][NP - 1] = fmaf(s[n][1], k0, x[n][blk][0][NP - 1]);
                        x[n][blk][1][0] = fmaf(s[n][2], k1, x[n][blk][1][0]);
                        x[n][blk][1][NP - 1] = fmaf(s[n][3], k1, x[n][blk][1][NP - 1]);
                    }
                }
            }
        }
        const int v0 = tile * KA_TILE;
        uint32_t bw[NT][2][GR][2];           // B columns of the weights
        const bool edge = masked || v0 + KA_TILE > count;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float top[NP];
#pragma unroll
            for (int i = 0; i < NP; i++) {
                top[i] = -INFINITY;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float& y = x[n][r >> 1][r & 1][i];
                    y *= sfac[n][i];
                    if (edge) {
                        const int v = v0 + r * 8 + g, rel = v - nsink;
                        const bool see = v < nsink ? v <= see_sink[n][i] : rel <= see_hi[n][i] && rel > see_lo[n][i];
                        if (!see || v >= count) y = -INFINITY;
                    }
                    top[i] = fmaxf(top[i], y);
                }
                top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 4));
                top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 8));
                top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 16));
            }
            if (__any_sync(0xffffffffu, top[0] > m[n][0] || top[NP - 1] > m[n][NP - 1])) {
                float c[NP];
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    const float mn = fmaxf(m[n][i], top[i]);
                    c[i] = m[n][i] == -INFINITY ? 1.0f : ka_exp2(m[n][i] - mn);   // nothing was summed before
                    l[n][i] *= c[i];
                    m[n][i] = mn;
                }
                // R is in units of 2^m of its column's pair
                const float c0 = __shfl_sync(0xffffffffu, c[0], g >> 1), c1 = __shfl_sync(0xffffffffu, c[NP - 1], g >> 1);
                R[n] *= PARTS == 2 || !(g & 1) ? c0 : c1;
                rinv[n] = KA_TOP / R[n];
            }
            // weights, and their move to B layout: tokens t + 4 i (i = 0..3) of
            // each 16, column g
            float pb_[2][4];
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const float ref = m[n][i] == -INFINITY ? 0.0f : m[n][i];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float& y = x[n][r >> 1][r & 1][i];
                    y = ka_exp2(y - ref);
                    l[n][i] += y;
                }
            }
#pragma unroll
            for (int blk = 0; blk < 2; blk++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int src = (t + 4 * (i & 1)) * 4 + (g >> 1);
                    const float y0 = __shfl_sync(0xffffffffu, x[n][blk][i >> 1][0], src);
                    if (PARTS == 2) {
                        pb_[blk][i] = y0;
                    } else {
                        const float y1 = __shfl_sync(0xffffffffu, x[n][blk][i >> 1][NP - 1], src);
                        pb_[blk][i] = (g & 1) ? y1 : y0;
                    }
                }
            // weight x value scale (a token of weight 0 may hold a NaN scale: masked for this pair)
            float w[2][GR][4], wtop = 0.0f;
#pragma unroll
            for (int blk = 0; blk < 2; blk++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int gr = 0; gr < GR; gr++) {
                        const float s = vs[(blk * 16 + t + 4 * i) * GR + gr];
                        w[blk][gr][i] = pb_[blk][i] != 0.0f ? pb_[blk][i] * s : 0.0f;
                        wtop = fmaxf(wtop, w[blk][gr][i]);
                    }
            wtop = fmaxf(wtop, __shfl_xor_sync(0xffffffffu, wtop, 1));
            wtop = fmaxf(wtop, __shfl_xor_sync(0xffffffffu, wtop, 2));
            if (__any_sync(0xffffffffu, wtop > R[n] || R[n] < KA_RMIN)) {
                const bool mine = wtop > R[n] || R[n] < KA_RMIN;
                const float rn = mine ? fmaxf(2.0f * wtop, KA_RMIN) : R[n];
                const float f = R[n] / rn;
                R[n] = rn;
                rinv[n] = KA_TOP / rn;
                const float f0 = __shfl_sync(0xffffffffu, f, 8 * t), f1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
                for (int i = 0; i < GR * 4; i++) {
                    acc[n][i][0] *= f0;
                    acc[n][i][1] *= f1;
                    acc[n][i][2] *= f0;
                    acc[n][i][3] *= f1;
                }
            }
#pragma unroll
            for (int blk = 0; blk < 2; blk++)
#pragma unroll
                for (int gr = 0; gr < GR; gr++) {
                    float* y = w[blk][gr];
                    const uint32_t b0 = ka_column<PARTS>(y[0] * rinv[n], y[1] * rinv[n], g & 1);
                    const uint32_t b1 = ka_column<PARTS>(y[2] * rinv[n], y[3] * rinv[n], g & 1);
                    bw[n][blk][gr][0] = b0;
                    bw[n][blk][gr][1] = b1;
                }
        }
        // values
#pragma unroll
        for (int blk = 0; blk < 2; blk++)
#pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                uint32_t wv[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = blk * 16 + t + 4 * i;
                    const int at = HD == 128 ? ((2 * gr + (g >> 2)) ^ (r & 2)) * 16 + 4 * (g & 3) : 4 * g;
                    wv[i] = *reinterpret_cast<const uint32_t*>(st + C::CODES + r * C::ROW + at);
                }
#pragma unroll
                for (int byte = 0; byte < 4; byte++) {
                    const uint32_t sel = (uint32_t)byte * 0x11u | (uint32_t)(4 + byte) * 0x1100u;
                    const uint32_t r01 = __byte_perm(wv[0], wv[1], sel), r23 = __byte_perm(wv[2], wv[3], sel);
                    const uint32_t a0 = ka_low(r01), a1 = ka_high(r01), a2 = ka_low(r23), a3 = ka_high(r23);
#pragma unroll
                    for (int n = 0; n < NT; n++)
                        ka_mma(acc[n][gr * 4 + byte], a0, a1, a2, a3, bw[n][blk][gr][0], bw[n][blk][gr][1]);
                }
            }
    }

    // ---- join: each warp's (m, l, sum) to shared memory, over the ring
    ka_wait<0>();
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem);                 // [warp][pair][HD]
    float* sm = so + KA_WARPS * PAIRS * HD;                     // [warp][pair]
    float* sl = sm + KA_WARPS * PAIRS;
    float* co = sl + KA_WARPS * PAIRS;                          // the block's own [pair][HD], [pair], [pair]
    float* cm = co + PAIRS * HD;
    float* cl = cm + PAIRS;
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const float back = R[n] * (1.0f / KA_TOP);
        const float e0 = __shfl_sync(0xffffffffu, back, 8 * t), e1 = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
        for (int i = 0; i < NP; i++) {
            float s = l[n][i];
            s += __shfl_xor_sync(0xffffffffu, s, 4);
            s += __shfl_xor_sync(0xffffffffu, s, 8);
            s += __shfl_xor_sync(0xffffffffu, s, 16);
            const int pair = n * (8 / PARTS) + (PARTS == 2 ? t : 2 * t + i);
            if (g == 0) {
                sm[warp * PAIRS + pair] = m[n][i];
                sl[warp * PAIRS + pair] = s;
            }
            float* o = so + (warp * PAIRS + pair) * HD;
#pragma unroll
            for (int k = 0; k < GR * 4; k++) {
                const int d = (k >> 2) * 64 + 8 * g + 2 * (k & 3);
                if (PARTS == 2) {
                    o[d] = (acc[n][k][0] + acc[n][k][1]) * e0;
                    o[d + 1] = (acc[n][k][2] + acc[n][k][3]) * e0;
                } else {
                    o[d] = acc[n][k][i] * (i ? e1 : e0);
                    o[d + 1] = acc[n][k][2 + i] * (i ? e1 : e0);
                }
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < PAIRS * HD; i += KA_WARPS * 32) {
        const int pair = i / HD;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < KA_WARPS; w++) mx = fmaxf(mx, sm[w * PAIRS + pair]);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        float o = 0.0f, s = 0.0f;
#pragma unroll
        for (int w = 0; w < KA_WARPS; w++) {
            const float f = ka_exp2(sm[w * PAIRS + pair] - ref);
            o = fmaf(so[w * PAIRS * HD + i], f, o);
            s = fmaf(sl[w * PAIRS + pair], f, s);
        }
        const int p = pair0 + pair;
        if (cluster == 1) {
            if (p < pairs)
                static_cast<T*>(a.out)[((long long)b * a.n_tokens + p / share) * a.ldo +
                                       (long long)(hk * share + p % share) * HD + i % HD] = dz_from_float<T>(o / s);
        } else {
            co[i] = o;
            if (i % HD == 0) {
                cm[pair] = mx;
                cl[pair] = s;
            }
        }
    }
    if (cluster == 1) return;
    // the blocks of the cluster each finish a share of the elements
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    const uint32_t co_s = (uint32_t)__cvta_generic_to_shared(co);
    auto remote = [&](int block, int index) {
        uint32_t at;
        float v;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(co_s + 4 * index), "r"(block));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
        return v;
    };
    for (int i = rank * KA_WARPS * 32 + threadIdx.x; i < PAIRS * HD; i += cluster * KA_WARPS * 32) {
        const int pair = i / HD, p = pair0 + pair;
        if (p >= pairs) break;
        float mx = -INFINITY;
        for (int c = 0; c < cluster; c++) mx = fmaxf(mx, remote(c, PAIRS * HD + pair));
        float o = 0.0f, s = 0.0f;
        for (int c = 0; c < cluster; c++) {
            const float f = ka_exp2(remote(c, PAIRS * HD + pair) - mx);
            o = fmaf(remote(c, i), f, o);
            s = fmaf(remote(c, PAIRS * HD + PAIRS + pair), f, s);
        }
        static_cast<T*>(a.out)[((long long)b * a.n_tokens + p / share) * a.ldo +
                               (long long)(hk * share + p % share) * HD + i % HD] = dz_from_float<T>(o / s);
    }
    // no block leaves while another may still read its shared memory
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}

template <int HD, int PARTS, int NT> constexpr int ka_smem() {
    constexpr int pairs = NT * 8 / PARTS;
    constexpr int join = ((KA_WARPS + 1) * pairs * HD + 2 * (KA_WARPS + 1) * pairs) * 4;
    return KaCfg<HD>::RING > join ? KaCfg<HD>::RING : join;
}

// Blocks of a cluster: one pass over the SMs' room with as many blocks as fit,
// while each warp still has a tile or two of the longest context that the ring
// allows.
static int ka_cluster(long long units, long long longest, int sms, int per_sm) {
    int best = 1;
    double cost = 1e30;
    for (int c = 1; c <= 8; c *= 2) {
        if (c > 1 && longest < (long long)c * KA_WARPS * KA_TILE) break;
        const double waves = (double)((units * c + (long long)sms * per_sm - 1) / ((long long)sms * per_sm));
        const double t = waves / c + 0.02 * c;
        if (t < cost) {
            cost = t;
            best = c;
        }
    }
    return best;
}

template <typename T, int HD, int PARTS, int NT>
static cudaError_t ka_launch(const Kv4AttnArgs& a, int device, int sms, cudaStream_t st) {
    auto* k = dz_kv4_attn_kernel<T, HD, PARTS, NT>;
    constexpr int smem = ka_smem<HD, PARTS, NT>(), pairs_per_block = NT * 8 / PARTS;
    static std::atomic<bool> ready[KA_DEVICES];
    if (device >= KA_DEVICES || !ready[device].load(std::memory_order_relaxed)) {
        const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (device < KA_DEVICES) ready[device].store(true, std::memory_order_relaxed);
    }
    const int pairs = a.n_tokens * (a.q_heads / a.c.kv_heads);
    const int blocks = (pairs + pairs_per_block - 1) / pairs_per_block;
    const long long units = (long long)a.c.batch * a.c.kv_heads * blocks;
    const long long ring = a.c.capacity - a.c.sinks;
    const long long longest = a.c.sinks + (a.window && a.window < ring ? a.window + a.n_tokens : ring);
    const int cluster = ka_cluster(units, longest, sms, NT == 1 ? 2 : 1);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * cluster));
    cfg.blockDim = dim3(KA_WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k, a, cluster, blocks);
}

template <typename T, int PARTS>
static cudaError_t ka_launch_t(const Kv4AttnArgs& a, int head_dim, int device, int sms, cudaStream_t st) {
    const bool one = a.n_tokens * (a.q_heads / a.c.kv_heads) <= 8 / PARTS;
    if (head_dim == 128)
        return one ? ka_launch<T, 128, PARTS, 1>(a, device, sms, st) : ka_launch<T, 128, PARTS, 2>(a, device, sms, st);
    return one ? ka_launch<T, 64, PARTS, 1>(a, device, sms, st) : ka_launch<T, 64, PARTS, 2>(a, device, sms, st);
}

cudaError_t dz_kv4_attn_launch(const Kv4AttnArgs& a, int type, int head_dim, int device, cudaStream_t st) {
    static std::atomic<int> sms[KA_DEVICES];   // SM count per device, looked up once
    int n = device < KA_DEVICES ? sms[device].load(std::memory_order_relaxed) : 0;
    if (!n) {
        const cudaError_t e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
        if (e != cudaSuccess) return e;
        if (device < KA_DEVICES) sms[device].store(n, std::memory_order_relaxed);
    }
    if (type == DZ_TYPE_F32) return ka_launch_t<float, 2>(a, head_dim, device, n, st);
    if (type == DZ_TYPE_F16) return ka_launch_t<__half, 2>(a, head_dim, device, n, st);
    return ka_launch_t<__nv_bfloat16, 1>(a, head_dim, device, n, st);
}

}  // namespace dz
