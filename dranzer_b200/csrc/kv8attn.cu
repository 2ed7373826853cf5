// Attention over the 8-bit paged caches (kv8.cuh): softmax(scale q . k) . v for
// the newest queries of every sequence, with fp32 sums and running statistics.
//
// A unit is one (sequence, key head) and up to 8 NT pairs (query token, query
// head). Tokens are the rows of the 16-bit MMAs (m16n8k16) of the scores, pairs
// their columns; elements of the head are the rows of those of the sums, pairs
// again their columns, so that few pairs leave few columns idle. Warps take
// tiles of 32 tokens of a unit in turn, a tile lying in one page, so that one
// scale for keys and one for values serve a whole tile. A lane loads 16 bytes
// of a token at a time straight into the MMAs' operands (elements and tokens
// may come in any order as long as the other operand follows it), without
// shared memory; the weights turn from the scores' result into the sums'
// operand by movmatrix. Codes become fp16 exactly, two at a time, by setting
// the exponent of 1024 above the byte and subtracting 1024 + 128.
//
// Queries are fp16 as they are, bf16 times a power of two of their row (its
// largest element in [2^13, 2^14)), fp32 the same in two fp16 parts; weights
// are taken times 2^15 in two fp16 parts. Scores of a tile take the page's key
// scale, the sums of a tile its value scale, both in fp32.
//
// Few units of long contexts go to clusters of blocks, many to a warp each
// (kv8_shape); the parts (maximum, sum of weights, sums) join at the end in
// shared memory, of a cluster through distributed shared memory.
#include <atomic>
#include <cooperative_groups.h>
#include <type_traits>

#include "dz_types.h"
#include "kv8.cuh"
#include "shim.cuh"

namespace dz {

namespace cg = cooperative_groups;

constexpr int KV8_TILE = 32;       // tokens that a warp takes at a time
constexpr int KV8_CLUSTER = 16;    // blocks of a cluster at most
constexpr int KV8_DEVICES = 64;    // devices whose launch state is kept
// Warps of a block: as many as their registers let an SM hold in one block.
template <int NT> struct Kv8Warps { static constexpr int N = NT == 1 ? 12 : 8; };

__device__ __forceinline__ void kv8_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The first product of a sum: no registers to clear.
__device__ __forceinline__ void kv8_mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint4 kv8_ld16(const int8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 kv8_ld8(const int8_t* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

// Bytes 2h and 2h + 1 of `biased` (code + 128) as two fp16 codes.
template <int H> __device__ __forceinline__ uint32_t kv8_widen(uint32_t biased) {
    const uint32_t x = __byte_perm(biased, 0x64646464u, H ? 0x4342 : 0x4140);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));      // 1152
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), off);
    return *reinterpret_cast<const uint32_t*>(&y);
}

__device__ __forceinline__ uint32_t kv8_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float kv8_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Rows and columns of an 8 x 8 matrix of 16-bit values exchanged: lane 4 r + c held (r, 2c), (r, 2c + 1).
__device__ __forceinline__ uint32_t kv8_turn(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Parts of a 16-bit query's element: one, of an fp32 one's: two.
template <typename T> struct Kv8Parts { static constexpr int N = 1; };
template <> struct Kv8Parts<float> { static constexpr int N = 2; };

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(Kv8Warps<NT>::N * 32, 1)
    dz_kv8_attn_kernel(const __grid_constant__ Kv8AttnArgs a, int team, int cluster, int blocks, int units) {
    constexpr int PARTS = Kv8Parts<T>::N, PAIRS = 8 * NT, WARPS = Kv8Warps<NT>::N;
    constexpr int STEPS = HD / 16;           // score MMAs over a head's elements, each of 4 bytes a lane and token
    constexpr int TILES = HD / 16;           // sum MMAs over a head's elements
    constexpr int COLS = HD / 8;             // a lane's elements of a token's value
    extern __shared__ __align__(16) float kv8_join[];                 // [warps][PAIRS][HD], then
    float2* stats = reinterpret_cast<float2*>(kv8_join + WARPS * PAIRS * HD);       // [warps][PAIRS] maximum, weights
    int* seens = reinterpret_cast<int*>(stats + WARPS * PAIRS);                     // [warps][PAIRS]
    // [warps][PARTS][NT][STEPS][32 lanes]: queries as B operands; registers for them would leave too few for the rest
    uint2* queries = reinterpret_cast<uint2*>(seens + WARPS * PAIRS);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = cluster > 1 ? (int)(blockIdx.x % (unsigned)cluster) : 0;
    const int unit = cluster > 1 ? blockIdx.x / cluster : blockIdx.x * (WARPS / team) + warp / team;
    const int warps = team * cluster, me = cluster > 1 ? rank * WARPS + warp : warp % team;
    const int share = a.q_heads / a.c.kv_heads, pairs = a.n_tokens * share;
    int b = 0, h = 0, r0 = 0, rows = 0;
    long long first = -1;
    if (unit < units) {
        const int blk = unit % blocks, bh = unit / blocks;
        h = bh % a.c.kv_heads;
        b = bh / a.c.kv_heads;
        r0 = blk * PAIRS;
        rows = min(PAIRS, pairs - r0);
        first = a.positions[b];
        if (kv8_skips(first)) rows = 0;
    }
    float o[TILES][NT][4];                   // elements COLS g + 2 i (0, 1) and + 1 (2, 3) of pairs 2 t, 2 t + 1
#pragma unroll
    for (int i = 0; i < TILES; i++)
#pragma unroll
        for (int n = 0; n < NT; n++) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.0f;
    // of pairs 8 n + 2 t + e: maximum, sum of this lane's weights, whether any token was seen
    float top[NT][2], sum[NT][2];
    int seen[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            top[n][e] = -INFINITY;
            sum[n][e] = 0.0f;
            seen[n][e] = 0;
        }
    if (rows > 0) {
        // what a pair sees: positions low..high, counted in 32 bits, nothing past the table
        const long long reach = (long long)a.c.table_pages * a.c.page;
        auto high_of = [&](int r) { return (int)min(first + min(r0 + r, pairs - 1) / share, reach); };
        auto low_of = [&](int r) {
            return a.window ? (int)min(max(0LL, first + min(r0 + r, pairs - 1) / share - a.window + 1), reach) : 0;
        };
        int high[NT][2], low[NT][2];
        float factor[NT][2];                 // what the pair's dot products take before the page's scale
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                high[n][e] = high_of(8 * n + 2 * t + e);
                low[n][e] = low_of(8 * n + 2 * t + e);
            }
        const int high_all = high_of(0), low_all = low_of(rows - 1);  // a tile within them is seen by every pair
        // queries as B operands: step s takes elements 64 (s / 4) + 16 t + 4 (s % 4) + 0..3 of pair 8 n + g
        uint2* qb = queries + (threadIdx.x >> 5) * (PARTS * NT * STEPS * 32) + lane;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int r = min(r0 + 8 * n + g, pairs - 1);
            const T* q = static_cast<const T*>(a.q) + ((long long)b * a.n_tokens + r / share) * a.ldq +
                         (h * share + r % share) * HD + 16 * t;
            float peak = 0.0f;
            bool bad = false;
#pragma unroll
            for (int s = 0; s < STEPS; s++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = dz_to_float(q[64 * (s / 4) + 4 * (s % 4) + e]);
                    peak = fmaxf(peak, fabsf(x));
                    bad |= !(fabsf(x) <= 3.402823466e38f);
                }
            float up = 1.0f, own = a.scale * 1.4426950408889634f;
            if (!std::is_same<T, __half>::value) {
                peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
                peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
                // 2^e that takes the largest to [2^13, 2^14), within fp32
                const int e = peak > 0.0f ? min(max(13 - (int)((__float_as_uint(peak) >> 23) & 255) + 127, -126), 126) : 0;
                up = __uint_as_float((unsigned)(e + 127) << 23);
                own *= __uint_as_float((unsigned)(127 - e) << 23);
            }
            bad |= __shfl_xor_sync(0xffffffffu, (int)bad, 1);
            bad |= __shfl_xor_sync(0xffffffffu, (int)bad, 2);
            if (bad) own = __int_as_float(0x7fc00000);
            factor[n][0] = __shfl_sync(0xffffffffu, own, 8 * t);      // of pair 2 t, which lanes 8 t.. hold
            factor[n][1] = __shfl_sync(0xffffffffu, own, 8 * t + 4);
#pragma unroll
            for (int s = 0; s < STEPS; s++) {
                uint32_t part[PARTS][2];
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const T* x = q + 64 * (s / 4) + 4 * (s % 4) + 2 * w;
                    const float u = dz_to_float(x[0]) * up, v = dz_to_float(x[1]) * up;
                    const uint32_t hi = kv8_half2(u, v);
                    part[0][w] = hi;
                    if (PARTS == 2) {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                        part[PARTS - 1][w] = kv8_half2(u - f.x, v - f.y);
                    }
                }
#pragma unroll
                for (int p = 0; p < PARTS; p++) qb[((p * NT + n) * STEPS + s) * 32] = make_uint2(part[p][0], part[p][1]);
            }
        }
        const int32_t* table = a.c.table + (long long)b * a.c.table_pages;
        const int shift = a.c.page == 64 ? 6 : 5;
        const int from = low_of(0), to = min(high_of(rows - 1), (int)reach - 1);
        const int t_first = from >> 5, t_last = to < from ? -1 : to >> 5;                 // tiles
        auto page_of = [&](int tile) {
            const int p = tile <= t_last ? table[tile >> (shift - 5)] : -1;
            return (unsigned)p < (unsigned)a.c.pages ? p : -1;
        };
        // where the tile's codes start, elements from the start of a code buffer
        auto place_of = [&](int page, int tile) {
            return ((long long)page * a.c.kv_heads + h) * (a.c.page * HD) + (shift == 6 ? (tile & 1) * (32 * HD) : 0);
        };
        uint32_t k[4][STEPS];                // the next tile's keys: token 8 i + g, 4 bytes a step
        auto load_k = [&](int page, int tile) {
            if (page < 0) return;
            const int8_t* p = a.c.k_codes + place_of(page, tile) + g * HD + t * 16;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int s = 0; s < STEPS / 4; s++)
                    *reinterpret_cast<uint4*>(&k[i][4 * s]) = kv8_ld16(p + i * (8 * HD) + s * 64);
        };
        int tile = t_first + me;
        int page = page_of(tile), next = page_of(tile + warps);
        load_k(page, tile);
        for (; tile <= t_last; tile += warps) {
            const int here = page;
            page = next;
            next = page_of(tile + 2 * warps);
            if (here < 0) {
                load_k(page, tile + warps);
                continue;
            }
            const float k_scale = a.c.k_scales[(long long)here * a.c.kv_heads + h];
            const float v_scale = a.c.v_scales[(long long)here * a.c.kv_heads + h];
            float s[2][NT][4];               // tokens 16 i + g (0, 1) and + 8 (2, 3), pairs 2 t, 2 t + 1
#pragma unroll
            for (int e = 0; e < STEPS; e++) {
                uint2 q[PARTS][NT];
#pragma unroll
                for (int p = 0; p < PARTS; p++)
#pragma unroll
                    for (int n = 0; n < NT; n++) q[p][n] = qb[((p * NT + n) * STEPS + e) * 32];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const uint32_t u = k[2 * i][e] ^ 0x80808080u, w = k[2 * i + 1][e] ^ 0x80808080u;
                    const uint32_t ka[4] = {kv8_widen<0>(u), kv8_widen<0>(w), kv8_widen<1>(u), kv8_widen<1>(w)};
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int p = 0; p < PARTS; p++) {
                            if (e == 0 && p == 0)
                                kv8_mma_first(s[i][n], ka, q[p][n].x, q[p][n].y);
                            else
                                kv8_mma(s[i][n], ka, q[p][n].x, q[p][n].y);
                        }
                }
            }
            // values: tokens 16 s + 2 t, + 1, + 8, + 9, elements COLS g .. COLS g + COLS - 1
            uint32_t v[2][4][COLS / 4];
            const int8_t* pv = a.c.v_codes + place_of(here, tile) + 2 * t * HD + g * COLS;
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int8_t* p = pv + (16 * s + (i & 1) + (i >> 1) * 8) * HD;
                    if (COLS == 16)
                        *reinterpret_cast<uint4*>(&v[s][i][0]) = kv8_ld16(p);
                    else
                        *reinterpret_cast<uint2*>(&v[s][i][0]) = kv8_ld8(p);
                }
            const int p0 = tile * KV8_TILE;
            const bool whole = p0 + KV8_TILE - 1 <= high_all && p0 >= low_all;
            float less[NT][2], shrink[NT][2], vs[NT][2];
            bool grown = false;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    // scores are f times the dot products, f >= 0 (their signs turned where it is not)
                    float f = k_scale * factor[n][e];
                    if (f < 0.0f) {
                        f = -f;
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            s[i][n][e] = -s[i][n][e];
                            s[i][n][2 + e] = -s[i][n][2 + e];
                        }
                    }
                    vs[n][e] = v_scale;
                    if (whole) {
                        seen[n][e] = 1;
                    } else {                 // value scale 0 where the pair sees nothing of the tile
                        int any = 0;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int p = p0 + 8 * i + g;
                            const bool sees = p <= high[n][e] && p >= low[n][e];
                            if (!sees) s[i / 2][n][i % 2 * 2 + e] = -INFINITY;
                            any |= sees;
                        }
                        any |= __shfl_xor_sync(0xffffffffu, any, 4);
                        any |= __shfl_xor_sync(0xffffffffu, any, 8);
                        any |= __shfl_xor_sync(0xffffffffu, any, 16);
                        if (!any) f = vs[n][e] = 0.0f;
                        seen[n][e] |= any;
                    }
                    f = f == 0.0f ? 1.17549435e-38f : f;       // hidden tokens stay at -inf
                    float m = fmaxf(fmaxf(s[0][n][e], s[0][n][2 + e]), fmaxf(s[1][n][e], s[1][n][2 + e]));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    m = fmaxf(top[n][e], m * f);
                    less[n][e] = (m == -INFINITY ? 0.0f : m) - 15.0f;            // weights times 2^15
                    shrink[n][e] = top[n][e] == m ? 1.0f : kv8_exp2(top[n][e] - m);
                    grown |= shrink[n][e] != 1.0f;
                    top[n][e] = m;
                    float w = 0.0f;
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            s[i][n][2 * j + e] = kv8_exp2(fmaf(s[i][n][2 * j + e], f, -less[n][e]));
                            w += s[i][n][2 * j + e];
                        }
                    sum[n][e] = fmaf(sum[n][e], shrink[n][e], w);
                }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int i = 0; i < TILES; i++)
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        o[i][n][0] *= shrink[n][0];
                        o[i][n][1] *= shrink[n][1];
                        o[i][n][2] *= shrink[n][0];
                        o[i][n][3] *= shrink[n][1];
                    }
            }
            // weights as B operands: tokens 16 i + 2 t, + 1 and + 8, + 9 of pair 8 n + g
            uint32_t wh[2][NT][2], wl[2][NT][2];
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const uint32_t hi = kv8_half2(s[i][n][2 * j], s[i][n][2 * j + 1]);
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                        wh[i][n][j] = kv8_turn(hi);
                        wl[i][n][j] = kv8_turn(kv8_half2(s[i][n][2 * j] - f.x, s[i][n][2 * j + 1] - f.y));
                    }
#pragma unroll
            for (int j4 = 0; j4 < COLS / 4; j4++) {
                // pairs of tokens side by side: bytes (token 0, token 1) of elements 4 j4 + 0, 1 and + 2, 3
                uint32_t lowb[2][2], highb[2][2];
#pragma unroll
                for (int st = 0; st < 2; st++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const uint32_t u = v[st][2 * c][j4] ^ 0x80808080u, w = v[st][2 * c + 1][j4] ^ 0x80808080u;
                        lowb[st][c] = __byte_perm(u, w, 0x5140);
                        highb[st][c] = __byte_perm(u, w, 0x7362);
                    }
#pragma unroll
                for (int e = 0; e < 2; e++) {                    // elements 4 j4 + 2 e, + 1
                    const int i = 2 * j4 + e;
                    float part[NT][4];
#pragma unroll
                    for (int st = 0; st < 2; st++) {
                        const uint32_t (&from2)[2] = e ? highb[st] : lowb[st];
                        const uint32_t va[4] = {kv8_widen<0>(from2[0]), kv8_widen<1>(from2[0]), kv8_widen<0>(from2[1]),
                                                kv8_widen<1>(from2[1])};
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            if (st == 0)
                                kv8_mma_first(part[n], va, wh[st][n][0], wh[st][n][1]);
                            else
                                kv8_mma(part[n], va, wh[st][n][0], wh[st][n][1]);
                            kv8_mma(part[n], va, wl[st][n][0], wl[st][n][1]);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        o[i][n][0] = fmaf(part[n][0], vs[n][0], o[i][n][0]);
                        o[i][n][1] = fmaf(part[n][1], vs[n][1], o[i][n][1]);
                        o[i][n][2] = fmaf(part[n][2], vs[n][0], o[i][n][2]);
                        o[i][n][3] = fmaf(part[n][3], vs[n][1], o[i][n][3]);
                    }
                }
            }
            load_k(page, tile + warps);
        }
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = 8 * n + 2 * t + e;
            float w = sum[n][e];
            w += __shfl_xor_sync(0xffffffffu, w, 4);
            w += __shfl_xor_sync(0xffffffffu, w, 8);
            w += __shfl_xor_sync(0xffffffffu, w, 16);
            float* at = kv8_join + (warp * PAIRS + r) * HD + g * COLS;
#pragma unroll
            for (int i = 0; i < TILES; i += 2)
                *reinterpret_cast<float4*>(at + 2 * i) =
                    make_float4(o[i][n][e], o[i][n][2 + e], o[i + 1][n][e], o[i + 1][n][2 + e]);
            if (g == 0) {
                stats[warp * PAIRS + r] = make_float2(top[n][e], w);
                seens[warp * PAIRS + r] = seen[n][e];
            }
        }
    if (cluster > 1)
        cg::this_cluster().sync();
    else
        __syncthreads();
    // outputs: the unit's rows over its team's lanes, or over all threads of a cluster
    const int wide = cluster > 1 ? cluster * WARPS * 32 : team * 32;
    const int self = cluster > 1 ? rank * (WARPS * 32) + (int)threadIdx.x : (warp % team) * 32 + lane;
    const int w0 = cluster > 1 ? 0 : warp / team * team;
    for (int x = self; x < rows * (HD / 4); x += wide) {
        const int r = x / (HD / 4), d = x % (HD / 4) * 4;
        float m = -INFINITY;
        int any = 0;
        for (int c = 0; c < cluster; c++) {
            const float2* st = cluster > 1 ? cg::this_cluster().map_shared_rank(stats, c) : stats;
            const int* sn = cluster > 1 ? cg::this_cluster().map_shared_rank(seens, c) : seens;
            for (int w = 0; w < team; w++) {
                m = fmaxf(m, st[(w0 + w) * PAIRS + r].x);
                any |= sn[(w0 + w) * PAIRS + r];
            }
        }
        float total = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int c = 0; c < cluster; c++) {
            const float2* st = cluster > 1 ? cg::this_cluster().map_shared_rank(stats, c) : stats;
            const float* jn = cluster > 1 ? cg::this_cluster().map_shared_rank(kv8_join, c) : kv8_join;
            for (int w = 0; w < team; w++) {
                const int at = (w0 + w) * PAIRS + r;
                const float2 s = st[at];
                const float f = s.x == -INFINITY ? 0.0f : s.x == m ? 1.0f : kv8_exp2(s.x - m);
                // a part that weighs nothing may still hold a NaN, which counts; one that saw nothing is all 0
                const float4 v = *reinterpret_cast<const float4*>(jn + at * HD + d);
                total = fmaf(s.y, f, total);
                y[0] = fmaf(v.x, f, y[0]);
                y[1] = fmaf(v.y, f, y[1]);
                y[2] = fmaf(v.z, f, y[2]);
                y[3] = fmaf(v.w, f, y[3]);
            }
        }
        const int pair = r0 + r;
        T* out = static_cast<T*>(a.out) + ((long long)b * a.n_tokens + pair / share) * a.ldo +
                 (h * share + pair % share) * HD + d;
#pragma unroll
        for (int i = 0; i < 4; i++) out[i] = dz_from_float<T>(any ? y[i] / total : 0.0f);
    }
    if (cluster > 1) cg::this_cluster().sync();      // no block ends while another reads its shared memory
}

// Clusters of 1..16 blocks of a kernel that a device holds at once (a cluster
// stays within one GPC, so that larger ones leave SMs idle; 0: it cannot hold
// one). Asked once per kernel and device.
struct Kv8Room {
    std::atomic<bool> known{false};
    std::atomic<int> clusters[KV8_CLUSTER + 1];
};

// Warps of a team and blocks of a cluster for `units` units of up to `longest`
// visible tokens: the least number of tiles that a warp works through one
// after the other, its start (as long as 4 tiles) and the joins (3 each) among
// them.
static void kv8_shape(const Kv8Room& room, int block_warps, long long units, long long longest, int* team, int* cluster) {
    const long long tiles = (longest + KV8_TILE - 1) / KV8_TILE;
    double best = 1e30;
    auto consider = [&](int w, int c) {
        const long long warps = (long long)w * c;
        const long long slots = (long long)room.clusters[c].load(std::memory_order_relaxed) * (block_warps / w);
        if (slots <= 0) return;
        const double waves = (double)((units + slots - 1) / slots), each = (double)((tiles + warps - 1) / warps);
        const double t = waves * (each + 4.0 + (warps > 1 ? 3.0 : 0.0) + (c > 1 ? 3.0 : 0.0));
        if (t < best) {
            best = t;
            *team = w;
            *cluster = c;
        }
    };
    for (int w = 1; w <= block_warps; w++)
        if (block_warps % w == 0) consider(w, 1);
    for (int c = 2; c <= KV8_CLUSTER && (long long)(c - 1) * block_warps < tiles; c++) consider(block_warps, c);
}

template <typename T, int HD, int NT>
static cudaError_t kv8_attn_t(const Kv8AttnArgs& a, long long longest, int device, cudaStream_t st) {
    static Kv8Room rooms[KV8_DEVICES];
    constexpr int PAIRS = 8 * NT, WARPS = Kv8Warps<NT>::N, smem = WARPS * PAIRS * (HD * 4 + (int)sizeof(float2) + 4 + HD * 2 * Kv8Parts<T>::N);
    const auto kernel = dz_kv8_attn_kernel<T, HD, NT>;
    Kv8Room& room = rooms[device];
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    if (!room.known.load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        for (int c = 1; c <= KV8_CLUSTER && e == cudaSuccess; c++) {
            cfg.gridDim = dim3(c);
            attr[0].val.clusterDim.x = c;
            int n = 0;
            e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
            room.clusters[c].store(n, std::memory_order_relaxed);
        }
        if (e != cudaSuccess) return e;
        room.known.store(true, std::memory_order_release);
    }
    const int pairs = a.n_tokens * (a.q_heads / a.c.kv_heads), blocks = (pairs + PAIRS - 1) / PAIRS;
    const long long units = (long long)a.c.batch * a.c.kv_heads * blocks;
    int team = 1, cluster = 1;
    kv8_shape(room, WARPS, units, a.window && a.window < longest ? a.window + a.n_tokens : longest, &team, &cluster);
    cfg.gridDim = dim3((unsigned)((units + WARPS / team - 1) / (WARPS / team) * cluster));
    attr[0].val.clusterDim.x = cluster;
    cfg.attrs = cluster > 1 ? attr : attr + 1;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, team, cluster, blocks, (int)units);
}

template <typename T>
static cudaError_t kv8_attn_h(const Kv8AttnArgs& a, long long longest, int head_dim, int device, cudaStream_t st) {
    const int pairs = a.n_tokens * (a.q_heads / a.c.kv_heads);
    if (head_dim == 128)
        return pairs <= 8 ? kv8_attn_t<T, 128, 1>(a, longest, device, st) : kv8_attn_t<T, 128, 2>(a, longest, device, st);
    if (pairs <= 8) return kv8_attn_t<T, 64, 1>(a, longest, device, st);
    return pairs <= 16 ? kv8_attn_t<T, 64, 2>(a, longest, device, st) : kv8_attn_t<T, 64, 4>(a, longest, device, st);
}

cudaError_t dz_kv8_attn_launch(const Kv8AttnArgs& a, long long longest, int type, int head_dim, int device, cudaStream_t st) {
    if (device < 0 || device >= KV8_DEVICES) return cudaErrorInvalidDevice;
    if (type == DZ_TYPE_F32) return kv8_attn_h<float>(a, longest, head_dim, device, st);
    if (type == DZ_TYPE_F16) return kv8_attn_h<__half>(a, longest, head_dim, device, st);
    return kv8_attn_h<__nv_bfloat16>(a, longest, head_dim, device, st);
}

}  // namespace dz
