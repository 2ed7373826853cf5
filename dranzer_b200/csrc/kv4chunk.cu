// Attention over the 4-bit ring caches (kv4.cuh) for many (query token, query
// head) pairs to a key head: chunks of tokens, prompts, wide sharing. In a
// translation unit of its own.
//
// A unit is one (sequence, key head) and 16 of its pairs, which are the rows of
// mma.m16n8k16; tokens are its columns, so the score accumulators become the
// weights' A operand in place and the codes are widened once for 16 pairs
// (kv4attn.cu has tokens as rows and at most 4 pairs to a unit, for decoding).
// Visible tokens go in tiles of 32 to a team of warps or a cluster of blocks,
// as there.
//
// Products. Codes become levels -7..7, exact in fp16 and bf16.
//   scores   A = queries in fp16, after a power of two that puts a row's
//            largest element in [2^14, 2^15): exact for 16-bit queries but for
//            what lies 2^-29 below it, two parts (hi = fp16(x), lo = fp16(x -
//            hi): 2^-24) for fp32. B = levels of K. Per 64-element group, times
//            the token's scale, in fp32.
//   values   A = weight x value scale in bf16 parts, whose range is fp32's: three
//            for fp32 (2^-27), two for 16-bit types (2^-18). B = levels of V.
// Sums, maxima and joins are fp32.
//
// Bound by instruction issue (2.2 a cycle per SM; the 16-bit MMAs take a
// third of the tensor pipe). On one B200, against kv4attn.cu's kernel: 8 x 4 key
// heads of 64, 16 tokens of 8 heads each over 4160 tokens, fp16, 42 us (91), fp32
// 56 us (122); key heads of 128, fp16, 77 us (162), fp32 98 us (230).
#include <cmath>

#include "kv4launch.cuh"
#include "shim.cuh"

namespace dz {

constexpr int KC_WARPS = KV4_WARPS;
constexpr int KC_TILE = KV4_TILE;
constexpr int KC_STAGES = 2;
constexpr int KC_ROWS = 16;      // pairs of a unit

template <int HD, int QP> struct KcCfg {
    static constexpr int ROW = HD / 2;
    static constexpr int GROUPS = HD / KV4_GROUP;
    static constexpr int CODES = KC_TILE * ROW;
    static constexpr int SCALES = KC_TILE * GROUPS * 4;
    static constexpr int STAGE = 2 * CODES + 2 * SCALES;
    static constexpr int QUERY = QP * (HD / 16) * 32 * 16;          // A fragments of a team's rows
    static constexpr int JOIN = (KC_ROWS * (HD + 4) + 2 * KC_ROWS) * 4;   // a warp's part: [row][HD + 4], m, l
    static constexpr int WARP = KC_STAGES * STAGE > JOIN ? KC_STAGES * STAGE : JOIN;
    static constexpr int BLOCK = KC_WARPS * (WARP + QUERY);   // (a cluster's block joins over its query area)
    static_assert(KC_WARPS * QUERY >= (KC_ROWS * HD + 2 * KC_ROWS) * 4 && WARP % 16 == 0, "");
};

__device__ __forceinline__ void kc_copy(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? 16 : 0;   // 0: the 16 bytes are zeroed
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n));
}
template <int BYTES> __device__ __forceinline__ void kc_copy_small(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? BYTES : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n));
}

__device__ __forceinline__ void kc_mma_f16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void kc_mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float kc_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// (w & mask) | base in one instruction: both constants stay in registers.
__device__ __forceinline__ uint32_t kc_mask_or(uint32_t w, uint32_t mask, uint32_t base) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(w), "r"(mask), "r"(base));
    return y;
}

// Levels of the nibbles at bits 0 and 16 (low) or 4 and 20 (high) of w as fp16
// pairs: 0x6400 is 1024, whose step is 1; or-ing a nibble in adds it or 16 x it.
// (A widely published way to widen 4-bit codes, here with their bias of 7.)
__device__ __forceinline__ uint32_t kc_low(uint32_t w) {
    const uint32_t x = kc_mask_or(w, 0x000F000Fu, 0x64006400u);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6407)));   // 1031
    return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ uint32_t kc_high(uint32_t w) {
    const uint32_t x = kc_mask_or(w, 0x00F000F0u, 0x64006400u);
    const __half2 y = __hfma2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x2C00)),    // 1/16
                              __half2half2(__ushort_as_half(0xD470)));                                          // -71
    return *reinterpret_cast<const uint32_t*>(&y);
}
// The same at bits 0 and 16 as bf16 pairs: 0x4300 is 128, whose step is 1.
__device__ __forceinline__ uint32_t kc_level(uint32_t w) {
    const uint32_t x = kc_mask_or(w, 0x000F000Fu, 0x43004300u);
    const __nv_bfloat162 y = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x),
                                     __bfloat162bfloat162(__ushort_as_bfloat16(0x4307)));                       // 135
    return *reinterpret_cast<const uint32_t*>(&y);
}

__device__ __forceinline__ uint32_t kc_pack_f16(float a, float b) {   // a in the low half
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t kc_pack_bf16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The chunk c (16 bytes) of row r lies at chunk c ^ kc_swizzle(r) (HD 128: two
// rows share the banks): K fragments read rows 0, 4, 1, 5 (and 2, 6, 3, 7) at
// once, V fragments rows 0..3 (and 4..7).
__device__ __forceinline__ int kc_swizzle(int r) { return ((r >> 1) ^ (r >> 2)) << 1 & 2; }

// Two blocks to an SM at head dimension 64. At 128 the accumulators leave room for
// one: two spilled 168 bytes a thread of 16-bit types, 8 x 4 key heads of 16 pairs
// over 4160 tokens 31 us against 22, 2 x 8 of 4 pairs over 130k 186 against 165.
template <typename T, int HD, int QP>   // QP: fp16 parts of a query
__global__ void __launch_bounds__(KC_WARPS * 32, HD == 64 ? 2 : 1) dz_kv4_chunk_kernel(
    const __grid_constant__ Kv4AttnArgs a, int team, int cluster, int pair_blocks, int units) {
    using C = KcCfg<HD, QP>;
    constexpr int GR = C::GROUPS, WP = QP == 2 ? 3 : 2;   // bf16 parts of a weight
    extern __shared__ __align__(16) uint8_t smem[];
    asm volatile("griddepcontrol.wait;" ::: "memory");    // launched while the kernel before ends
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % cluster, tw = warp % team;
    int unit = blockIdx.x / cluster * (KC_WARPS / team) + warp / team;
    if (unit >= units) return;               // whole teams of a single block
    const int pb = unit % pair_blocks;
    unit /= pair_blocks;
    const int hk = unit % a.c.kv_heads, b = unit / a.c.kv_heads;
    const long long first = a.positions[b] + a.pos_add;
    if (kv4_skips(first)) return;   // the whole team, or cluster, leaves
    const int share = a.q_heads / a.c.kv_heads, pairs = share * a.n_tokens, pair0 = pb * KC_ROWS;

    // ---- the virtual index v = 0..count-1 runs over the sinks, then over positions lo, lo + 1, ...
    const long long ring = a.c.capacity - a.c.sinks, last = first + a.n_tokens - 1;
    const int j_lo = pair0 / share, j_hi = min((pair0 + KC_ROWS - 1) / share, a.n_tokens - 1);
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

    uint8_t* my = smem + warp * C::WARP;
    const uint32_t my_s = (uint32_t)__cvta_generic_to_shared(my);
    auto slot_of = [&](int v) {
        if (v < nsink) return v;
        const unsigned s = (unsigned)(v - nsink) + (unsigned)start;   // both below 2^31
        return (int)(s >= (unsigned)cap ? s - (unsigned)iring : s);
    };
    constexpr int CH = C::ROW / 16, RPI = 32 / CH;            // chunks of a row, rows of one pass over the lanes
    auto issue = [&](int tile, int stage) {
        const uint32_t s = my_s + stage * C::STAGE;
        const int v0 = tile * KC_TILE, s0 = slot_of(v0);
        // whole, neither across the sinks' end nor round the ring: one run of slots
        if (v0 + KC_TILE <= count && (v0 >= nsink || v0 + KC_TILE <= nsink) && s0 + KC_TILE <= cap) {
            const uint8_t* k = kc + (long long)s0 * C::ROW + lane * 16;
            const uint8_t* v = vc + (long long)s0 * C::ROW + lane * 16;
            const uint32_t ds = s + 2 * C::CODES + lane * GR * 4;
#pragma unroll
            for (int i = 0; i < KC_TILE / RPI; i++) {
                const int r = lane / CH + i * RPI, c = lane % CH;
                const uint32_t d = s + r * C::ROW + (HD == 128 ? c ^ kc_swizzle(r) : c) * 16;
                kc_copy(d, k + i * 512, true);
                kc_copy(d + C::CODES, v + i * 512, true);
            }
            kc_copy_small<GR * 4>(ds, ksc + ((long long)s0 + lane) * GR, true);
            kc_copy_small<GR * 4>(ds + C::SCALES, vsc + ((long long)s0 + lane) * GR, true);
            return;
        }
#pragma unroll
        for (int i = 0; i < KC_TILE / RPI; i++) {
            const int r = lane / CH + i * RPI, c = lane % CH, v = v0 + r;
            const long long off = (long long)(v < count ? slot_of(v) : 0) * C::ROW + c * 16;
            const uint32_t d = s + r * C::ROW + (HD == 128 ? c ^ kc_swizzle(r) : c) * 16;
            kc_copy(d, kc + off, v < count);
            kc_copy(d + C::CODES, vc + off, v < count);
        }
        const bool valid = v0 + lane < count;
        const long long off = (long long)(valid ? slot_of(v0 + lane) : 0) * GR;
        const uint32_t ds = s + 2 * C::CODES + lane * GR * 4;
        kc_copy_small<GR * 4>(ds, ksc + off, valid);
        kc_copy_small<GR * 4>(ds + C::SCALES, vsc + off, valid);
    };
    const int ntiles = (count + KC_TILE - 1) / KC_TILE, step = team * cluster;
    const int tile0 = rank * team + tw;
    if (tile0 < ntiles) issue(tile0, 0);
    asm volatile("cp.async.commit_group;");

    // ---- query fragments of the team, in shared memory: rows g and g + 8, lane t's
    // elements in the order in which a code word's nibbles become B registers.
    // Every warp of the team needs a row's factor, one warp writes the fragments.
    uint4* qs = reinterpret_cast<uint4*>(smem + KC_WARPS * C::WARP + (warp - tw) * C::QUERY);
    float sfac[2];                           // scale x log2 e / the row's power of two
    {
        uint32_t frag[QP][HD / 16][4];
#pragma unroll
        for (int h = 0; h < 2; h++) {        // rows g, g + 8
            const int pair = pair0 + g + 8 * h;
            const bool live = pair < pairs;
            const T* q = static_cast<const T*>(a.q) +
                         ((long long)b * a.n_tokens + (live ? pair / share : 0)) * a.ldq +
                         (long long)(hk * share + (live ? pair % share : 0)) * HD + 16 * t;
            float x[GR * 16], top = 0.0f;
            bool bad = false;
#pragma unroll
            for (int i = 0; i < GR * 16; i++) {
                x[i] = live ? dz_to_float(q[(i / 16) * 64 + i % 16]) : 0.0f;
                top = fmaxf(top, fabsf(x[i]));
                bad |= !(fabsf(x[i]) <= 3.402823466e38f);
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            bad = __any_sync(0xfu << (lane & 28), bad);
            // 2^(14 - e) for top in [2^e, 2^(e + 1)), its exponent kept in a normal float's range
            const int e = min(141 - (int)(__float_as_uint(top) >> 23), 126);
            const float f = __int_as_float((127 + e) << 23);
            sfac[h] = bad ? __int_as_float(0x7fc00000) : a.scale * 1.4426950408889634f * __int_as_float((127 - e) << 23);
#pragma unroll
            for (int w = 0; w < GR * 2; w++)   // word w of the lane: elements 8 w .. 8 w + 7 of its x
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    // k-step 2 w + k: nibbles 0 4 | 1 5 (k = 0), 2 6 | 3 7 (k = 1)
                    float y[4] = {x[8 * w + 2 * k] * f, x[8 * w + 2 * k + 4] * f, x[8 * w + 2 * k + 1] * f,
                                  x[8 * w + 2 * k + 5] * f};
#pragma unroll
                    for (int p = 0; p < QP; p++) {
                        const uint32_t b0 = kc_pack_f16(y[0], y[1]), b1 = kc_pack_f16(y[2], y[3]);
                        frag[p][2 * w + k][h] = b0;
                        frag[p][2 * w + k][2 + h] = b1;
                        const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&b0));
                        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&b1));
                        y[0] -= u.x; y[1] -= u.y; y[2] -= v.x; y[3] -= v.y;
                    }
                }
        }
        if (tw == 0)
#pragma unroll
            for (int p = 0; p < QP; p++)
#pragma unroll
                for (int k = 0; k < HD / 16; k++)
                    qs[(p * (HD / 16) + k) * 32 + lane] = make_uint4(frag[p][k][0], frag[p][k][1], frag[p][k][2], frag[p][k][3]);
    }
    const int bar = 1 + warp / team;
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(team * 32) : "memory");

    // ---- what rows g and g + 8 see
    int see_sink[2], see_hi[2], see_lo[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int pair = min(pair0 + g + 8 * h, pairs - 1);
        const long long pos = first + pair / share;
        see_sink[h] = (int)min(pos, (long long)INT32_MAX);
        see_hi[h] = (int)max(-1LL, pos - lo);
        see_lo[h] = a.window ? (int)max(-1LL, pos - a.window - lo) : -1;
    }
    // tiles of later positions that every row sees: rel in (all_lo, all_hi]
    const int all_hi = (int)max(-1LL, first + j_lo - lo);
    const int all_lo = a.window ? (int)max(-1LL, first + j_hi - a.window - lo) : -1;

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float acc[GR * 8][4];                    // n-tile 8 gr + j: elements 64 gr + 16 t + j and + 8 of rows g, g + 8
#pragma unroll
    for (int i = 0; i < GR * 8; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) acc[i][r] = 0.0f;

    int stage = 0;
    for (int tile = tile0; tile < ntiles; tile += step) {
        asm volatile("cp.async.wait_group 0;");
        __syncwarp();
        if (tile + step < ntiles) issue(tile + step, stage ^ 1);
        asm volatile("cp.async.commit_group;");
        const uint8_t* st = my + stage * C::STAGE;
        stage ^= 1;
        const float* ks = reinterpret_cast<const float*>(st + 2 * C::CODES);
        const float* vs = ks + KC_TILE * GR;

        // ---- scores: n-tile i, column n is token 8 i + n / 2 + 4 (n % 2); this lane's columns 2t, 2t + 1 are
        // tokens 8 i + t and 8 i + t + 4
        float x[4][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = 8 * i + (g >> 1) + 4 * (g & 1);
#pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                const int at = HD == 128 ? ((2 * gr + (t >> 1)) ^ kc_swizzle(r)) * 16 + 8 * (t & 1) : 8 * t;
                const uint2 w = *reinterpret_cast<const uint2*>(st + r * C::ROW + at);
                float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const uint32_t c = (u ? w.y : w.x) >> (8 * k), b0 = kc_low(c), b1 = kc_high(c);
#pragma unroll
                        for (int p = 0; p < QP; p++)
                            kc_mma_f16(s, qs[(p * (HD / 16) + 4 * gr + 2 * u + k) * 32 + lane], b0, b1);
                    }
                const float k0 = ks[(8 * i + t) * GR + gr], k1 = ks[(8 * i + t + 4) * GR + gr];
#pragma unroll
                for (int c = 0; c < 4; c++) x[i][c] = gr ? fmaf(s[c], c & 1 ? k1 : k0, x[i][c]) : s[c] * (c & 1 ? k1 : k0);
            }
        }
        const int v0 = tile * KC_TILE, rel0 = v0 - nsink;
        const bool edge = v0 + KC_TILE > count || !(rel0 > all_lo && v0 >= nsink && rel0 + KC_TILE - 1 <= all_hi);
        // ---- softmax: rows g (h = 0) and g + 8
        bool grows = false;
        float top[2];
        unsigned hidden = 0;
        if (edge) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int h = c >> 1, v = v0 + 8 * i + t + 4 * (c & 1), rel = v - nsink;
                    const bool see = v < nsink ? v <= see_sink[h] : rel <= see_hi[h] && rel > see_lo[h];
                    x[i][c] = see && v < count ? x[i][c] * sfac[h] : -INFINITY;
                    if (!see || v >= count) hidden |= 1u << (4 * i + c);
                }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) x[i][c] *= sfac[c >> 1];
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            top[h] = fmaxf(fmaxf(fmaxf(x[0][2 * h], x[0][2 * h + 1]), fmaxf(x[1][2 * h], x[1][2 * h + 1])),
                           fmaxf(fmaxf(x[2][2 * h], x[2][2 * h + 1]), fmaxf(x[3][2 * h], x[3][2 * h + 1])));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
            grows |= top[h] > m[h];
        }
        if (__any_sync(0xffffffffu, grows)) {
            float f[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float mn = fmaxf(m[h], top[h]);
                f[h] = m[h] == -INFINITY ? 0.0f : kc_exp2(m[h] - mn);   // nothing was summed before
                l[h] *= f[h];
                m[h] = mn;
            }
#pragma unroll
            for (int i = 0; i < GR * 8; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) acc[i][r] *= f[r >> 1];
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float ref = m[h] == -INFINITY ? 0.0f : m[h];
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    float& y = x[i][2 * h + c];
                    y = kc_exp2(y - ref);
                    l[h] += y;
                }
        }
        // a token that another row sees may hold a NaN scale: its weight is marked by its sign, and makes no product
        // (a token that is seen and whose weight is 0 makes one: its NaN counts)
        if (edge) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if (hidden >> (4 * i + c) & 1) x[i][c] = -0.0f;
        }
        // ---- values: 16 tokens (two n-tiles of scores) at a time
#pragma unroll
        for (int gr = 0; gr < GR; gr++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                // weight x value scale: rows g, g + 8 (h) of tokens t, t + 4, then of t + 8, t + 12 (i)
                float ws[2][2][2];
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const float s = vs[(16 * j + 8 * i + t + 4 * c) * GR + gr];
                        ws[i][0][c] = x[2 * j + i][c] * s;
                        ws[i][1][c] = x[2 * j + i][2 + c] * s;
                    }
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int c = 0; c < 4; c++)
                            if (__float_as_uint(x[2 * j + i][c]) == 0x80000000u) ws[i][c >> 1][c & 1] = 0.0f;
                }
                uint32_t wa[WP][4];
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int p = 0; p < WP; p++) {
                            const uint32_t q = kc_pack_bf16(ws[i][h][0], ws[i][h][1]);
                            wa[p][2 * i + h] = q;
                            if (p + 1 < WP) {
                                ws[i][h][0] -= __uint_as_float(q << 16);
                                ws[i][h][1] -= __uint_as_float(q & 0xffff0000u);
                            }
                        }
                uint32_t w[4];               // word g of tokens t, t + 4, t + 8, t + 12
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = 16 * j + t + 4 * i;
                    const int at = HD == 128 ? ((2 * gr + (g >> 2)) ^ kc_swizzle(r)) * 16 + 4 * (g & 3) : 4 * g;
                    w[i] = *reinterpret_cast<const uint32_t*>(st + C::CODES + r * C::ROW + at);
                }
#pragma unroll
                for (int byte = 0; byte < 4; byte++) {
                    const uint32_t sel = (uint32_t)byte * 0x11u | (uint32_t)(4 + byte) * 0x1100u;
                    const uint32_t r0 = __byte_perm(w[0], w[1], sel), r1 = __byte_perm(w[2], w[3], sel);
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const uint32_t b0 = kc_level(r0 >> (4 * k)), b1 = kc_level(r1 >> (4 * k));
#pragma unroll
                        for (int p = 0; p < WP; p++) kc_mma_bf16(acc[8 * gr + 2 * byte + k], wa[p], b0, b1);
                    }
                }
            }
    }

    // ---- the warp's sums; then the team's, then the cluster's
    asm volatile("cp.async.wait_group 0;");
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; h++) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    auto store_out = [&](int p, int d, float v) {
        static_cast<T*>(a.out)[((long long)b * a.n_tokens + p / share) * a.ldo +
                               (long long)(hk * share + p % share) * HD + d] = dz_from_float<T>(v);
    };
    if (team * cluster == 1) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int p = pair0 + g + 8 * h;
            if (p >= pairs) continue;
            const float inv = 1.0f / l[h];
            T* o = static_cast<T*>(a.out) + ((long long)b * a.n_tokens + p / share) * a.ldo +
                   (long long)(hk * share + p % share) * HD + 16 * t;
#pragma unroll
            for (int gr = 0; gr < GR; gr++)
#pragma unroll
                for (int d = 0; d < 16; d++)
                    o[64 * gr + d] = dz_from_float<T>(acc[8 * gr + d % 8][2 * h + d / 8] * inv);
        }
        return;
    }
    constexpr int OS = HD + 4;
    float* so = reinterpret_cast<float*>(my);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float* o = so + (g + 8 * h) * OS + 16 * t;
#pragma unroll
        for (int gr = 0; gr < GR; gr++)
#pragma unroll
            for (int d = 0; d < 16; d += 4)
                *reinterpret_cast<float4*>(o + 64 * gr + d) =
                    make_float4(acc[8 * gr + d % 8][2 * h + d / 8], acc[8 * gr + d % 8 + 1][2 * h + d / 8],
                                acc[8 * gr + d % 8 + 2][2 * h + d / 8], acc[8 * gr + d % 8 + 3][2 * h + d / 8]);
        if (t == 0) {
            so[KC_ROWS * OS + g + 8 * h] = m[h];
            so[KC_ROWS * OS + KC_ROWS + g + 8 * h] = l[h];
        }
    }
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(team * 32) : "memory");
    constexpr int MINE = C::WARP / 4;
    const float* t0 = reinterpret_cast<const float*>(smem) + (warp - tw) * MINE;
    float* co = reinterpret_cast<float*>(smem + KC_WARPS * C::WARP);   // a cluster's block: [row][HD], m, l, over its queries
    for (int i = tw * 32 + lane; i < KC_ROWS * HD; i += team * 32) {
        const int row = i / HD, d = i % HD, p = pair0 + row;
        if (p >= pairs) break;
        float mx = -INFINITY;
        for (int w = 0; w < team; w++) mx = fmaxf(mx, t0[w * MINE + KC_ROWS * OS + row]);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        float o = 0.0f, s = 0.0f;
        for (int w = 0; w < team; w++) {
            const float* q = t0 + w * MINE;
            const float f = kc_exp2(q[KC_ROWS * OS + row] - ref);
            o = fmaf(q[row * OS + d], f, o);
            s = fmaf(q[KC_ROWS * OS + KC_ROWS + row], f, s);
        }
        if (cluster == 1) {
            store_out(p, d, o / s);
        } else {
            co[i] = o;
            if (d == 0) {
                co[KC_ROWS * HD + row] = mx;
                co[KC_ROWS * HD + KC_ROWS + row] = s;
            }
        }
    }
    if (cluster == 1) return;
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    const uint32_t co_s = (uint32_t)__cvta_generic_to_shared(co);
    auto remote = [&](int block, int index) {
        uint32_t at;
        float v;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(co_s + 4 * index), "r"(block));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
        return v;
    };
    for (int i = rank * KC_WARPS * 32 + threadIdx.x; i < KC_ROWS * HD; i += cluster * KC_WARPS * 32) {
        const int row = i / HD, p = pair0 + row;
        if (p >= pairs) break;
        float mx = -INFINITY;
        for (int c = 0; c < cluster; c++) mx = fmaxf(mx, remote(c, KC_ROWS * HD + row));
        float o = 0.0f, s = 0.0f;
        for (int c = 0; c < cluster; c++) {
            const float f = kc_exp2(remote(c, KC_ROWS * HD + row) - mx);
            o = fmaf(remote(c, i), f, o);
            s = fmaf(remote(c, KC_ROWS * HD + KC_ROWS + row), f, s);
        }
        store_out(p, i % HD, o / s);
    }
    // no block leaves while another may still read its shared memory
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}

template <typename T, int HD, int QP>
static cudaError_t kc_launch(const Kv4AttnArgs& a, int device, cudaStream_t st) {
    static Kv4Room rooms[KV4_DEVICES];
    return kv4_launch(dz_kv4_chunk_kernel<T, HD, QP>, rooms, a, KC_ROWS, KcCfg<HD, QP>::BLOCK, device, st);
}

cudaError_t dz_kv4_chunk_launch(const Kv4AttnArgs& a, int type, int head_dim, int device, cudaStream_t st) {
    if (type == DZ_TYPE_F32)
        return head_dim == 128 ? kc_launch<float, 128, 2>(a, device, st) : kc_launch<float, 64, 2>(a, device, st);
    if (type == DZ_TYPE_F16)
        return head_dim == 128 ? kc_launch<__half, 128, 1>(a, device, st) : kc_launch<__half, 64, 1>(a, device, st);
    return head_dim == 128 ? kc_launch<__nv_bfloat16, 128, 1>(a, device, st)
                           : kc_launch<__nv_bfloat16, 64, 1>(a, device, st);
}

}  // namespace dz
