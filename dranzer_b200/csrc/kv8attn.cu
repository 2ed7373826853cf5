// Attention over the 8-bit paged caches (kv8.cuh): softmax(scale q . k) . v for
// the newest queries of every sequence, with fp32 sums and running statistics.
//
// A unit is one (sequence, key head) and up to 16 pairs (query token, query
// head); pairs are the rows of 16-bit MMAs (m16n8k16), tokens the columns of
// the scores, head elements the columns of the sums. Warps take tiles of 32
// tokens of a unit in turn, a tile lying in one page, so that one scale for
// keys and one for values serve a whole tile. A lane loads 16 bytes of a token
// at a time straight into the MMAs' operands (elements and columns may come in
// any order as long as the other operand follows it): no shared memory, no
// transposition. Codes become fp16 exactly, two at a time, by setting the
// exponent of 1024 above the byte and subtracting 1024 + 128.
//
// Queries are fp16 as they are, bf16 times a power of two of their row (its
// largest element in [2^13, 2^14)), fp32 the same in two fp16 parts; weights
// are taken times 2^15 in two fp16 parts. Scores of a tile take the page's key
// scale, the sums of a tile its value scale, both in fp32.
//
// Few units of long contexts go to clusters of blocks, many to a warp each
// (kv4_shape); the parts (maximum, sum of weights, sums) join at the end in
// shared memory, of a cluster through distributed shared memory.
#include <atomic>
#include <cooperative_groups.h>
#include <type_traits>

#include "dz_types.h"
#include "kv4launch.cuh"
#include "kv8.cuh"
#include "shim.cuh"

namespace dz {

namespace cg = cooperative_groups;

constexpr int KV8_TILE = 32;       // tokens that a warp takes at a time
constexpr int KV8_PAIRS = 16;      // rows of a unit

__device__ __forceinline__ void kv8_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

// Parts of a 16-bit query's element: one, of an fp32 one's: two.
template <typename T> struct Kv8Parts { static constexpr int N = 1; };
template <> struct Kv8Parts<float> { static constexpr int N = 2; };

template <typename T, int HD>
__global__ void __launch_bounds__(KV4_WARPS * 32, 1) dz_kv8_attn_kernel(const __grid_constant__ Kv8AttnArgs a, int team,
                                                                       int cluster, int blocks, int units) {
    constexpr int PARTS = Kv8Parts<T>::N;
    constexpr int STEPS = HD / 16;           // MMAs over a head's elements, each of 4 bytes a lane
    constexpr int COLS = HD / 8;             // MMAs over a token's values
    extern __shared__ __align__(16) float kv8_join[];                 // [warps][16][HD], then stats
    float2* stats = reinterpret_cast<float2*>(kv8_join + KV4_WARPS * KV8_PAIRS * HD);   // [warps][16] maximum, weights
    int* seens = reinterpret_cast<int*>(stats + KV4_WARPS * KV8_PAIRS);                 // [warps][16]
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = cluster > 1 ? (int)(blockIdx.x % (unsigned)cluster) : 0;
    const int unit = cluster > 1 ? blockIdx.x / cluster : blockIdx.x * (KV4_WARPS / team) + warp / team;
    const int warps = team * cluster, me = cluster > 1 ? rank * KV4_WARPS + warp : warp % team;
    const int share = a.q_heads / a.c.kv_heads, pairs = a.n_tokens * share;
    int b = 0, h = 0, r0 = 0, rows = 0;
    long long first = -1;
    if (unit < units) {
        const int blk = unit % blocks, bh = unit / blocks;
        h = bh % a.c.kv_heads;
        b = bh / a.c.kv_heads;
        r0 = blk * KV8_PAIRS;
        rows = min(KV8_PAIRS, pairs - r0);
        first = a.positions[b];
        if (kv8_skips(first)) rows = 0;
    }
    float o[COLS][4];
#pragma unroll
    for (int j = 0; j < COLS; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
    int seen[2] = {0, 0};
    if (rows > 0) {
        // the rows' positions, and the unit's range of tokens
        const long long reach = (long long)a.c.table_pages * a.c.page;
        const long long i_lo = first + r0 / share, i_hi = first + (r0 + rows - 1) / share;
        const long long pos[2] = {first + min(r0 + g, pairs - 1) / share, first + min(r0 + g + 8, pairs - 1) / share};
        const long long from = a.window ? max(0LL, i_lo - a.window + 1) : 0, to = min(i_hi, reach - 1);
        // queries as A operands: step s takes elements 64 (s / 4) + 16 t + 4 (s % 4) + 0..3
        uint32_t qa[PARTS][STEPS][4];
        float factor[2];
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const int r = min(r0 + g + half * 8, pairs - 1);
            const T* q = static_cast<const T*>(a.q) + ((long long)b * a.n_tokens + r / share) * a.ldq +
                         (h * share + r % share) * HD;
            float x[STEPS][4];
            float peak = 0.0f;
            bool bad = false;
#pragma unroll
            for (int s = 0; s < STEPS; s++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[s][e] = dz_to_float(q[64 * (s / 4) + 16 * t + 4 * (s % 4) + e]);
                    peak = fmaxf(peak, fabsf(x[s][e]));
                    bad |= !(fabsf(x[s][e]) <= 3.402823466e38f);
                }
            factor[half] = a.scale * 1.4426950408889634f;
            float up = 1.0f;
            if (!std::is_same<T, __half>::value) {
                peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
                peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
                // 2^e that takes the largest to [2^13, 2^14), within fp32
                const int e = peak > 0.0f ? min(max(13 - (int)((__float_as_uint(peak) >> 23) & 255) + 127, -126), 126) : 0;
                up = __uint_as_float((unsigned)(e + 127) << 23);
                factor[half] *= __uint_as_float((unsigned)(127 - e) << 23);
            }
            bad |= __shfl_xor_sync(0xffffffffu, (int)bad, 1);
            bad |= __shfl_xor_sync(0xffffffffu, (int)bad, 2);
            if (bad) factor[half] = __int_as_float(0x7fc00000);
#pragma unroll
            for (int s = 0; s < STEPS; s++)
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const float u = x[s][2 * w] * up, v = x[s][2 * w + 1] * up;
                    const uint32_t hi = kv8_half2(u, v);
                    qa[0][s][half + 2 * w] = hi;
                    if (PARTS == 2) {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                        qa[PARTS - 1][s][half + 2 * w] = kv8_half2(u - f.x, v - f.y);
                    }
                }
        }
        const int32_t* table = a.c.table + (long long)b * a.c.table_pages;
        const int shift = a.c.page == 64 ? 6 : 5;
        const int t_first = to < from ? 0 : (int)(from >> 5), t_last = to < from ? -1 : (int)(to >> 5);   // tiles
        auto page_of = [&](int tile) {
            const int p = tile <= t_last ? table[tile >> (shift - 5)] : -1;
            return (unsigned)p < (unsigned)a.c.pages ? p : -1;
        };
        // where the tile's codes start, elements from the start of a code buffer
        auto place_of = [&](int page, int tile) {
            return ((long long)page * a.c.kv_heads + h) * (a.c.page * HD) + (shift == 6 ? (tile & 1) * (32 * HD) : 0);
        };
        uint32_t k[4][STEPS];                // this tile's keys: token 8 i + g, 4 bytes a step
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
            const float k_scale = a.c.k_scales[(long long)here * a.c.kv_heads + h];
            const float v_scale = a.c.v_scales[(long long)here * a.c.kv_heads + h];
            float s[4][4];                   // scores: rows g (0, 1) and g + 8 (2, 3), tokens 8 i + 2 t, + 1
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
#pragma unroll
                for (int e = 0; e < STEPS; e++) {
                    const uint32_t biased = k[i][e] ^ 0x80808080u;
                    const uint32_t b0 = kv8_widen<0>(biased), b1 = kv8_widen<1>(biased);
                    kv8_mma(s[i], qa[0][e], b0, b1);
                    if (PARTS == 2) kv8_mma(s[i], qa[PARTS - 1][e], b0, b1);
                }
            }
            load_k(page, tile + warps);
            const float f[2] = {k_scale * factor[0], k_scale * factor[1]};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[i][0] *= f[0];
                s[i][1] *= f[0];
                s[i][2] *= f[1];
                s[i][3] *= f[1];
            }
            // value scales of the rows: 0 where a row sees nothing of the tile
            float vs[2] = {v_scale, v_scale};
            const long long p0 = (long long)tile * KV8_TILE;
            if (p0 + KV8_TILE - 1 <= i_lo && p0 + KV8_TILE <= reach && (!a.window || p0 > i_hi - a.window)) {
                seen[0] = seen[1] = 1;       // every row sees the whole tile
            } else {
                int any[2] = {0, 0};
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const long long p = p0 + 8 * i + 2 * t + (e & 1), at = pos[e >> 1];
                        const bool sees = p <= at && (!a.window || p > at - a.window);
                        if (!sees) s[i][e] = -INFINITY;
                        any[e >> 1] |= sees;
                    }
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    any[r] |= __shfl_xor_sync(0xffffffffu, any[r], 1);
                    any[r] |= __shfl_xor_sync(0xffffffffu, any[r], 2);
                    if (!any[r]) vs[r] = 0.0f;
                    seen[r] |= any[r];
                }
            }
            float less[2], shrink[2];
#pragma unroll
            for (int r = 0; r < 2; r++) {
                float m = top[r];
#pragma unroll
                for (int i = 0; i < 4; i++) m = fmaxf(m, fmaxf(s[i][2 * r], s[i][2 * r + 1]));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                less[r] = (m == -INFINITY ? 0.0f : m) - 15.0f;       // weights times 2^15
                shrink[r] = top[r] == m ? 1.0f : kv8_exp2(top[r] - m);
                top[r] = m;
            }
            uint32_t hi[4][2], lo[4][2];
#pragma unroll
            for (int r = 0; r < 2; r++) {
                sum[r] *= shrink[r];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float w0 = kv8_exp2(s[i][2 * r] - less[r]), w1 = kv8_exp2(s[i][2 * r + 1] - less[r]);
                    sum[r] += w0 + w1;
                    hi[i][r] = kv8_half2(w0, w1);
                    const float2 w = __half22float2(*reinterpret_cast<const __half2*>(&hi[i][r]));
                    lo[i][r] = kv8_half2(w0 - w.x, w1 - w.y);
                }
            }
            if (__any_sync(0xffffffffu, shrink[0] != 1.0f || shrink[1] != 1.0f)) {
#pragma unroll
                for (int j = 0; j < COLS; j++) {
                    o[j][0] *= shrink[0];
                    o[j][1] *= shrink[0];
                    o[j][2] *= shrink[1];
                    o[j][3] *= shrink[1];
                }
            }
            const uint32_t wh[2][4] = {{hi[0][0], hi[0][1], hi[1][0], hi[1][1]}, {hi[2][0], hi[2][1], hi[3][0], hi[3][1]}};
            const uint32_t wl[2][4] = {{lo[0][0], lo[0][1], lo[1][0], lo[1][1]}, {lo[2][0], lo[2][1], lo[3][0], lo[3][1]}};
#pragma unroll
            for (int j4 = 0; j4 < COLS / 4; j4++) {
                // pairs of tokens side by side: bytes (token 0, token 1) of elements 4 j4 + 0, 1 and + 2, 3
                uint32_t low[2][2], high[2][2];
#pragma unroll
                for (int st = 0; st < 2; st++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const uint32_t u = v[st][2 * c][j4] ^ 0x80808080u, w = v[st][2 * c + 1][j4] ^ 0x80808080u;
                        low[st][c] = __byte_perm(u, w, 0x5140);
                        high[st][c] = __byte_perm(u, w, 0x7362);
                    }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int st = 0; st < 2; st++) {
                        const uint32_t (&from4)[2] = e < 2 ? low[st] : high[st];
                        const uint32_t b0 = e % 2 ? kv8_widen<1>(from4[0]) : kv8_widen<0>(from4[0]);
                        const uint32_t b1 = e % 2 ? kv8_widen<1>(from4[1]) : kv8_widen<0>(from4[1]);
                        kv8_mma(part, wh[st], b0, b1);
                        kv8_mma(part, wl[st], b0, b1);
                    }
                    const int j = 4 * j4 + e;
                    o[j][0] = fmaf(part[0], vs[0], o[j][0]);
                    o[j][1] = fmaf(part[1], vs[0], o[j][1]);
                    o[j][2] = fmaf(part[2], vs[1], o[j][2]);
                    o[j][3] = fmaf(part[3], vs[1], o[j][3]);
                }
            }
        }
    }
    // a lane's sums stand for elements COLS (2 t) + j and COLS (2 t + 1) + j of rows g and g + 8
#pragma unroll
    for (int r = 0; r < 2; r++) {
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
        float* to = kv8_join + (warp * KV8_PAIRS + g + 8 * r) * HD + 2 * t * COLS;
#pragma unroll
        for (int j = 0; j < COLS; j += 4) {
            *reinterpret_cast<float4*>(to + j) =
                make_float4(o[j][2 * r], o[j + 1][2 * r], o[j + 2][2 * r], o[j + 3][2 * r]);
            *reinterpret_cast<float4*>(to + COLS + j) =
                make_float4(o[j][2 * r + 1], o[j + 1][2 * r + 1], o[j + 2][2 * r + 1], o[j + 3][2 * r + 1]);
        }
        if (t == 0) {
            stats[warp * KV8_PAIRS + g + 8 * r] = make_float2(top[r], sum[r]);
            seens[warp * KV8_PAIRS + g + 8 * r] = seen[r];
        }
    }
    if (cluster > 1)
        cg::this_cluster().sync();
    else
        __syncthreads();
    // outputs: the unit's rows over its team's lanes, or over all threads of a cluster
    const int wide = cluster > 1 ? cluster * KV4_WARPS * 32 : team * 32;
    const int self = cluster > 1 ? rank * (KV4_WARPS * 32) + (int)threadIdx.x : (warp % team) * 32 + lane;
    const int w0 = cluster > 1 ? 0 : warp / team * team;
    for (int x = self; x < rows * (HD / 4); x += wide) {
        const int r = x / (HD / 4), d = x % (HD / 4) * 4;
        float m = -INFINITY;
        int any = 0;
        for (int c = 0; c < cluster; c++) {
            const float2* st = cluster > 1 ? cg::this_cluster().map_shared_rank(stats, c) : stats;
            const int* sn = cluster > 1 ? cg::this_cluster().map_shared_rank(seens, c) : seens;
            for (int w = 0; w < team; w++) {
                m = fmaxf(m, st[(w0 + w) * KV8_PAIRS + r].x);
                any |= sn[(w0 + w) * KV8_PAIRS + r];
            }
        }
        float total = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int c = 0; c < cluster; c++) {
            const float2* st = cluster > 1 ? cg::this_cluster().map_shared_rank(stats, c) : stats;
            const float* jn = cluster > 1 ? cg::this_cluster().map_shared_rank(kv8_join, c) : kv8_join;
            for (int w = 0; w < team; w++) {
                const int at = (w0 + w) * KV8_PAIRS + r;
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

template <typename T, int HD>
static cudaError_t kv8_attn_t(const Kv8AttnArgs& a, long long longest, int device, cudaStream_t st) {
    static Kv4Room rooms[KV4_DEVICES];
    constexpr int smem = KV4_WARPS * KV8_PAIRS * (HD * 4 + (int)sizeof(float2) + 4);
    const auto kernel = dz_kv8_attn_kernel<T, HD>;
    Kv4Room& room = rooms[device];
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(KV4_WARPS * 32);
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
        for (int c = 1; c <= KV4_CLUSTER && e == cudaSuccess; c++) {
            cfg.gridDim = dim3(c);
            attr[0].val.clusterDim.x = c;
            int n = 0;
            e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
            room.clusters[c].store(n, std::memory_order_relaxed);
        }
        if (e != cudaSuccess) return e;
        room.known.store(true, std::memory_order_release);
    }
    const int pairs = a.n_tokens * (a.q_heads / a.c.kv_heads), blocks = (pairs + KV8_PAIRS - 1) / KV8_PAIRS;
    const long long units = (long long)a.c.batch * a.c.kv_heads * blocks;
    int team = 1, cluster = 1;
    kv4_shape(room, units, a.window && a.window < longest ? a.window + a.n_tokens : longest, &team, &cluster);
    cfg.gridDim = dim3((unsigned)((units + KV4_WARPS / team - 1) / (KV4_WARPS / team) * cluster));
    attr[0].val.clusterDim.x = cluster;
    cfg.attrs = cluster > 1 ? attr : attr + 1;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, team, cluster, blocks, (int)units);
}

template <typename T>
static cudaError_t kv8_attn_h(const Kv8AttnArgs& a, long long longest, int head_dim, int device, cudaStream_t st) {
    return head_dim == 128 ? kv8_attn_t<T, 128>(a, longest, device, st) : kv8_attn_t<T, 64>(a, longest, device, st);
}

cudaError_t dz_kv8_attn_launch(const Kv8AttnArgs& a, long long longest, int type, int head_dim, int device, cudaStream_t st) {
    if (device < 0 || device >= KV4_DEVICES) return cudaErrorInvalidDevice;
    if (type == DZ_TYPE_F32) return kv8_attn_h<float>(a, longest, head_dim, device, st);
    if (type == DZ_TYPE_F16) return kv8_attn_h<__half>(a, longest, head_dim, device, st);
    return kv8_attn_h<__nv_bfloat16>(a, longest, head_dim, device, st);
}

}  // namespace dz
