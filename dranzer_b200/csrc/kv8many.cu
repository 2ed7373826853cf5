// Attention over the 8-bit paged caches of many queries (kv8attn.cuh): drafted
// tokens of grouped heads, chunks of a prompt.
//
// A block takes up to 128 pairs (query token, query head) of one sequence and
// key head, the lanes of tensor memory, and tiles of 128 tokens in turn, which
// the blocks of a cluster share. A tile's codes come by TMA, two tiles ahead in
// boxes of 32 tokens, and are widened to fp16 in shared memory once for all
// pairs (warps of kv8attn.cu widen them for 16 pairs at a time, a quarter of
// their instructions): keys are the K-major operand of the scores' MMAs, values,
// as they lie, the N-major one of the sums'. Scores stay in tensor memory; a
// thread reads those of its pair with 64 of the tokens, and writes weights back
// as the fp16 operand of the sums' MMAs in the scores' place. Each half of the
// threads keeps a maximum, a sum and the sums of values of its tokens; they and
// the cluster's blocks' join at the end.
//
// 32 x 128 pairs over 4112 tokens of heads of 64 in fp16 take 38 us (49 in warps
// of 16 pairs), 512 tokens of 32 heads of 128 in bf16 over 8512 positions 244 (560),
// 284 TFLOP/s. Bound by the chain of a tile (about 3 us of a block alone: a fifth
// widening, a sixth the scores' maximum, two fifths weights, a fifth sums), not by
// a unit; only the second block of an SM, with heads of 64, fills its gaps. Packed
// fp32 operations gained nothing.
//
// Queries are fp16 times a power of two of their row (its largest element in
// [2^13, 2^14)), fp32 ones in two parts; codes are fp16 exactly; weights are taken
// times 2^15 in two fp16 parts (kv8attn.cu has what these hold, and why). The
// pages' key scales meet the scores in fp32. Where two pages of different value
// scales share a thread's 64 tokens, the weights take these over one scale, which
// the tile's sums take in fp32: that of the page whose largest weight x scale is
// larger, times that weight, so that what counts keeps its bits whatever the
// scales are.
#include <cooperative_groups.h>
#include <type_traits>

#include "dz_types.h"
#include "kv8attn.cuh"
#include "tcgen05.cuh"

namespace dz {

namespace cg = cooperative_groups;

constexpr int KV8M_THREADS = 256;  // two halves of 128
constexpr int KV8M_PAIRS = 128;
constexpr int KV8M_KEYS = 128;     // tokens of a tile
constexpr int KV8M_CHUNKS = KV8M_KEYS / KV8_TILE;

template <typename T, int HD> struct Kv8Many {
    static constexpr int PARTS = std::is_same<T, float>::value ? 2 : 1;      // fp16 parts of a query's element
    static constexpr int PANEL = 128 * 128;                // 128 rows of 64 fp16, 128-byte swizzle
    static constexpr int PANELS = HD / 64;
    static constexpr int BOX = KV8_TILE * HD;              // codes of 32 tokens
    static constexpr int STAGE = 2 * KV8M_CHUNKS * BOX;    // keys, values of a tile
    static constexpr int WIDE = 2 * STAGE;                 // where widened keys, then values begin
    static constexpr int JOIN = 2 * KV8M_PAIRS * HD * 4;   // both halves' sums, over what comes before the queries
    static constexpr int QUERIES = WIDE + 2 * PANELS * PANEL;
    static constexpr int STATS = QUERIES + PARTS * PANELS * PANEL;           // [2][128] maximum, weights
    static constexpr int FACTORS = STATS + 2 * KV8M_PAIRS * 8;               // [128] what a pair's dot products take
    static constexpr int BARS = FACTORS + KV8M_PAIRS * 4;
    static constexpr int NEED = 1024 + BARS + 64;
    // two blocks to an SM with heads of 64, one with 128, which leaves no block of a product beside it: the tensor
    // memory that an SM's blocks hold at a time stays within its 512 columns, and no allocation waits
    static constexpr int COLUMNS = HD == 64 ? 256 : 512;
    static constexpr int SMEM = HD == 64 ? NEED : NEED > 190 * 1024 ? NEED : 190 * 1024;
    static_assert(JOIN <= QUERIES && SMEM <= (HD == 64 ? 113 : 227) * 1024, "shared memory");
};

__device__ __forceinline__ void kv8m_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// The first operand in tensor memory.
__device__ __forceinline__ void kv8m_mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// N-major operand, 128-byte swizzle: groups of 8 tokens 1024 bytes apart, panels of 64 elements of the head a panel apart.
__device__ __forceinline__ uint64_t kv8m_desc_values(uint32_t saddr, uint32_t panel) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)(panel >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 | (uint64_t)1u << 46 |
           (uint64_t)2u << 61;
}
__device__ __forceinline__ void kv8m_store8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void kv8m_load16(uint32_t taddr, float (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
          "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr)
        : "memory");
}

// Sixteen codes as fp16 in their order.
__device__ __forceinline__ void kv8m_widen(const uint4& in, uint4 (&out)[2]) {
    const uint32_t w[4] = {in.x, in.y, in.z, in.w};
    uint32_t y[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t near = __byte_perm(w[i], 0u, 0x4140), far = __byte_perm(w[i], 0u, 0x4342);    // bytes 0, 1 and 2, 3 as 16 bits
        y[2 * i] = kv8_widen<false>(near);
        y[2 * i + 1] = kv8_widen<false>(far);
    }
    out[0] = make_uint4(y[0], y[1], y[2], y[3]);
    out[1] = make_uint4(y[4], y[5], y[6], y[7]);
}

template <typename T, int HD>
__global__ void __launch_bounds__(KV8M_THREADS, HD == 64 ? 2 : 1)
    dz_kv8_many_kernel(const __grid_constant__ Kv8AttnArgs a, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, int cluster, int blocks) {
    using B = Kv8Many<T, HD>;
    extern __shared__ __align__(1024) uint8_t kv8m_raw[];
    uint8_t* sm = kv8m_raw + ((1024u - (dz_smem_addr(kv8m_raw) & 1023u)) & 1023u);
    float2* stats = reinterpret_cast<float2*>(sm + B::STATS);
    float* factors = reinterpret_cast<float*>(sm + B::FACTORS);
    uint64_t* codes_bar = reinterpret_cast<uint64_t*>(sm + B::BARS);         // [2] a stage's codes have come
    uint64_t* scores_bar = codes_bar + 2;
    uint64_t* sums_bar = scores_bar + 1;                                     // [2] of the halves
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sums_bar + 2);
    volatile int* failed = reinterpret_cast<int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp >> 2, r = (warp & 3) * 32 + lane;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 5; i++) dz_mbar_init(&codes_bar[i]);
        *failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // tensor memory only after the kernel before has ended: its blocks may still want theirs
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dz_smem_addr(tmem_slot)),
                     "r"((uint32_t)B::COLUMNS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const int rank = (int)(blockIdx.x % (unsigned)cluster), unit = (int)(blockIdx.x / (unsigned)cluster);
    const int share = a.q_heads / a.c.kv_heads, pairs = a.n_tokens * share;
    const int blk = unit % blocks, h = unit / blocks % a.c.kv_heads, b = unit / blocks / a.c.kv_heads;
    const int r0 = blk * KV8M_PAIRS;
    const long long first = a.positions[b];
    // queries: HD / 8 lanes have a row, a warp 16; all on their way before the position is needed
    constexpr int LANES = HD / 8, STEP = 32 / LANES, SETS = 16 / STEP;
    union Row {
        T e[8];
        uint4 w[sizeof(T) / 2];
        __device__ Row() {}
    } own[SETS];
    const bool wide = ((uintptr_t)a.q | (uintptr_t)(a.ldq * (long long)sizeof(T))) % 16 == 0;
#pragma unroll
    for (int n = 0; n < SETS; n++) {
        const int pair = min(r0 + warp * 16 + n * STEP + lane / LANES, pairs - 1);
        const T* q = static_cast<const T*>(a.q) + ((long long)b * a.n_tokens + pair / share) * a.ldq + (h * share + pair % share) * HD +
                     8 * (lane % LANES);
        if (wide) {
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; k++) own[n].w[k] = reinterpret_cast<const uint4*>(q)[k];
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) own[n].e[k] = q[k];
        }
    }
    const int rows = kv8_skips(first) ? 0 : min(KV8M_PAIRS, pairs - r0);
    const bool busy = (warp & 3) * 32 < rows;                // the warp has pairs
    // what a pair sees: positions low..high, counted in 32 bits, nothing past the table
    const long long reach = (long long)a.c.table_pages * a.c.page;
    auto high_of = [&](int i) { return (int)min(first + min(r0 + i, pairs - 1) / share, reach); };
    auto low_of = [&](int i) {
        return a.window ? (int)min(max(0LL, first + min(r0 + i, pairs - 1) / share - a.window + 1), reach) : 0;
    };
    int tiles = 0, start = 0, high_all = -1, low_all = 0, high = -1, low = 0;     // start: the first tile's first box
    if (rows > 0) {
        const int from = low_of(0), to = min(high_of(rows - 1), (int)reach - 1);
        start = from >> 5;
        if (to >= from) tiles = ((to >> 5) - start) / KV8M_CHUNKS + 1;
        high_all = high_of(0);
        low_all = low_of(rows - 1);
        high = high_of(r);
        low = low_of(r);
    }
    const int mine = tiles > rank ? (tiles - rank - 1) / cluster + 1 : 0;         // of this block: rank, rank + cluster, ...
    const int shift = a.c.page == 64 ? 1 : 0, boxes = a.c.table_pages << shift;
    const int32_t* table = a.c.table + (long long)b * a.c.table_pages;
    // the table's entry of a box, which is looked at only when it is needed, and the page it names, -1: none
    auto entry = [&](int tile, int chunk) {
        const int box = start + (rank + tile * cluster) * KV8M_CHUNKS + chunk;
        return tile < mine && box < boxes ? table[box >> shift] : -1;
    };
    auto page_of = [&](int raw) { return (unsigned)raw < (unsigned)a.c.pages ? raw : -1; };
    const bool copies = warp == KV8M_THREADS / 32 - 1;       // the warp that fetches codes
    const bool elected = (warp == 0 || copies) && ug_elect();
    int ahead[2];                            // its entries of the next two tiles, lanes 0..3
#pragma unroll
    for (int n = 0; n < 2; n++) ahead[n] = copies && lane < KV8M_CHUNKS ? entry(n, lane) : -1;
    int raw[2] = {entry(0, 2 * half), entry(0, 2 * half + 1)};       // the half's two boxes of the next tile
    // a row's power of two takes its largest element to [2^13, 2^14)
#pragma unroll
    for (int n = 0; n < SETS; n++) {
        const int row = warp * 16 + n * STEP + lane / LANES, c = lane % LANES;
        float x[8], peak = 0.0f;
        bool bad = false;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            x[k] = dz_to_float(own[n].e[k]);
            peak = fmaxf(peak, fabsf(x[k]));
            bad |= !(fabsf(x[k]) <= 3.402823466e38f);
        }
#pragma unroll
        for (int off = LANES / 2; off >= 1; off >>= 1) {
            peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, off));
            bad |= __shfl_xor_sync(0xffffffffu, (int)bad, off);
        }
        // 2^e in two factors within fp32
        const int e = peak > 0.0f ? 13 - (int)((__float_as_uint(peak) >> 23) & 255) + 127 : 0;
        const int e0 = min(max(e, -126), 126), e1 = e - e0;
        const float up0 = __uint_as_float((unsigned)(e0 + 127) << 23), up1 = __uint_as_float((unsigned)(e1 + 127) << 23);
        if (c == 0)
            factors[row] = bad ? __int_as_float(0x7fc00000)
                               : a.scale * 1.4426950408889634f * __uint_as_float((unsigned)(127 - e0) << 23) *
                                     __uint_as_float((unsigned)(127 - e1) << 23);
        uint32_t w[B::PARTS][4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float u = bad ? 0.0f : x[2 * k] * up0 * up1, v = bad ? 0.0f : x[2 * k + 1] * up0 * up1;
            w[0][k] = kv8_half2(u, v);
            if (B::PARTS == 2) {
                const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&w[0][k]));
                w[B::PARTS - 1][k] = kv8_half2(u - hi.x, v - hi.y);
            }
        }
#pragma unroll
        for (int part = 0; part < B::PARTS; part++)
            *reinterpret_cast<uint4*>(sm + B::QUERIES + (part * B::PANELS + c / 8) * B::PANEL + row * 128 + ((c ^ row) & 7) * 16) =
                make_uint4(w[part][0], w[part][1], w[part][2], w[part][3]);
    }
    // a tile's codes on their way, by one warp
    auto fetch = [&](int tile, int raw) {
        const int page = page_of(raw), box = start + (rank + tile * cluster) * KV8M_CHUNKS;
        uint8_t* to = sm + (tile & 1) * B::STAGE;
        const int present = __popc(__ballot_sync(0xffffffffu, lane < KV8M_CHUNKS && page >= 0));
        if (elected) dz_mbar_expect_tx(&codes_bar[tile & 1], 2 * present * B::BOX);
#pragma unroll
        for (int i = 0; i < KV8M_CHUNKS; i++) {
            const int p = __shfl_sync(0xffffffffu, page, i);
            const int row = h * a.c.page + (shift ? ((box + i) & 1) * KV8_TILE : 0);
            if (p >= 0 && elected) {
                kv8_copy(to + i * B::BOX, &tm_k, row, p, &codes_bar[tile & 1]);
                kv8_copy(to + (KV8M_CHUNKS + i) * B::BOX, &tm_v, row, p, &codes_bar[tile & 1]);
            }
        }
    };
    ug_fence_before();
    __syncthreads();                                         // barriers, tensor memory, factors
    if (copies)
#pragma unroll
        for (int n = 0; n < 2; n++)
            if (n < mine) fetch(n, ahead[n]);
    // the half's two boxes of a tile: pages, scales
    const float *k_scales = a.c.k_scales + h, *v_scales = a.c.v_scales + h;
    int page[2];
    float ks[2], vs[2];
    auto scales = [&] {
#pragma unroll
        for (int c = 0; c < 2; c++) {
            page[c] = page_of(raw[c]);
            ks[c] = page[c] >= 0 ? k_scales[(long long)page[c] * a.c.kv_heads] : 0.0f;
            vs[c] = page[c] >= 0 ? v_scales[(long long)page[c] * a.c.kv_heads] : 0.0f;
        }
    };
    scales();
    raw[0] = entry(1, 2 * half);
    raw[1] = entry(1, 2 * half + 1);
    ahead[0] = copies && lane < KV8M_CHUNKS ? entry(2, lane) : -1;
    float o[HD];
#pragma unroll
    for (int i = 0; i < HD; i++) o[i] = 0.0f;
    float top = -INFINITY, sum = 0.0f;
    bool seen = false;                       // any token, whatever its score
    ug_fence_after();
    const uint32_t tmem = *tmem_slot;
    const float factor = factors[r];
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t scores = lanes + (uint32_t)(64 * half), sums = lanes + (uint32_t)(128 + HD * half);
    constexpr uint32_t F32 = 1u << 4, N_MAJOR = 1u << 16, M128 = (uint32_t)(128 >> 4) << 24;
    constexpr uint32_t scores_desc = F32 | M128 | (uint32_t)(KV8M_KEYS >> 3) << 17, sums_desc = F32 | M128 | N_MAJOR | (uint32_t)(HD >> 3) << 17;
    int i = 0;
    bool ok = true;
    for (; i < mine; i++) {
        const int stage = i & 1;
        if (!dz_mbar_wait(&codes_bar[stage], (uint32_t)((i >> 1) & 1))) ok = false;
        // widen: a thread has 16 codes of a token at a time, its warp 32 tokens' (a box that is not there holds any codes)
#pragma unroll
        for (int v = 0; v < 2; v++)
#pragma unroll
            for (int j = 0; j < HD / 32; j++) {
                const int piece = warp + 8 * j, box = piece & 3, at = piece >> 2;      // 16-byte chunk `at` of a box's rows
                const int turn = HD == 128 ? lane & 7 : lane >> 1 & 3;
                const uint4 in = *reinterpret_cast<const uint4*>(sm + stage * B::STAGE + (v * KV8M_CHUNKS + box) * B::BOX + lane * HD +
                                                                 ((at ^ turn) * 16));
                uint4 out[2];
                kv8m_widen(in, out);
                uint8_t* to = sm + B::WIDE + (v * B::PANELS + at / 4) * B::PANEL + (box * 32 + lane) * 128;
                *reinterpret_cast<uint4*>(to + ((at * 2 ^ lane) & 7) * 16) = out[0];
                *reinterpret_cast<uint4*>(to + ((at * 2 + 1 ^ lane) & 7) * 16) = out[1];
            }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        ug_fence_before();
        __syncthreads();
        if (warp == 0) {
            ug_fence_after();
            const uint64_t q = ug_desc_kmajor(dz_smem_addr(sm + B::QUERIES)), k = ug_desc_kmajor(dz_smem_addr(sm + B::WIDE));
            if (elected) {
#pragma unroll
                for (int part = 0; part < B::PARTS; part++)
#pragma unroll
                    for (int kk = 0; kk < HD / 16; kk++) {
                        const uint32_t at = (uint32_t)(kk / 4 * B::PANEL + kk % 4 * 32) >> 4;
                        kv8m_mma(tmem, q + ((uint32_t)(part * B::PANELS * B::PANEL) >> 4) + at, k + at, scores_desc, part || kk ? 1u : 0u);
                    }
                ug_commit(scores_bar);
            }
            __syncwarp();
        } else if (copies && i + 2 < mine) {                 // the stage's codes have been read
            fetch(i + 2, ahead[0]);
            ahead[0] = lane < KV8M_CHUNKS ? entry(i + 3, lane) : -1;
        }
        float shrink = 1.0f, vt = 0.0f;
        if (busy) {
            if (!dz_mbar_wait(scores_bar, (uint32_t)(i & 1))) ok = false;
            ug_fence_after();
            // without a sign: a tile may pass the end of the longest table
            const unsigned p0 = (unsigned)(start + (rank + i * cluster) * KV8M_CHUNKS) * KV8_TILE + 64u * half;
            float f[2], box[2], m = top;         // box: each one's largest score
            // a box that every pair sees whole, of scales that leave the scores' order, needs no look at its tokens
            bool plain[2];
            int lo[2], hi[2];                // what this pair sees of it; a page that is not there: nothing
            unsigned sign[2];                // scores are f times the dot products, f > 0: signs turned where the scales' differ
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const unsigned p = p0 + c * KV8_TILE;
                sign[c] = (ks[c] < 0.0f) != (a.scale < 0.0f) ? 0x80000000u : 0u;
                plain[c] = page[c] >= 0 && p + KV8_TILE - 1 <= (unsigned)high_all && p >= (unsigned)low_all && !sign[c];
                lo[c] = page[c] >= 0 ? (int)((unsigned)low - p) : KV8_TILE;
                hi[c] = page[c] >= 0 ? (int)((unsigned)high - p) : -1;
                f[c] = fabsf(ks[c] * factor);
                f[c] = f[c] == 0.0f ? 1.17549435e-38f : f[c];                // hidden tokens stay at -inf
                int32_t raw[32];
                ug_tmem_ld32(scores + (uint32_t)(c * 32), raw);
                float most[2] = {-INFINITY, -INFINITY};
                if (plain[c]) {
                    seen = true;
#pragma unroll
                    for (int j = 0; j < 32; j++) most[j & 1] = fmaxf(most[j & 1], __int_as_float(raw[j]));
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        most[j & 1] = fmaxf(most[j & 1], j >= lo[c] && j <= hi[c] ? __uint_as_float((unsigned)raw[j] ^ sign[c]) : -INFINITY);
                    if (max(lo[c], 0) > min(hi[c], KV8_TILE - 1)) {          // nothing, whatever the scales are
                        f[c] = 1.17549435e-38f;
                        vs[c] = 0.0f;
                    } else {
                        seen = true;
                    }
                }
                box[c] = fmaxf(most[0], most[1]) * f[c];
                m = fmaxf(m, box[c]);
            }
            const float less = 15.0f - (m == -INFINITY ? 0.0f : m);          // weights times 2^15
            shrink = top == m ? 1.0f : kv8_exp2(top - m);
            top = m;
            // the scale that the tile's sums take: where the boxes' differ, the one that the largest weight x scale sets (no
            // smaller than 2^-100 of the larger scale, so that quotients stay in range)
            vt = fmaxf(fabsf(vs[0]), fabsf(vs[1]));
            if (fabsf(vs[0]) != fabsf(vs[1]) && fminf(fabsf(vs[0]), fabsf(vs[1])) > 0.0f) {
                float most = vt * 0x1p-100f;
#pragma unroll
                for (int c = 0; c < 2; c++) most = fmaxf(most, box[c] == -INFINITY ? 0.0f : fabsf(vs[c]) * kv8_exp2(box[c] - m));
                if (most > 0.0f) vt = most;
            }
            float total[2] = {0.0f, 0.0f};
            // weights of a box, 16 tokens at a time, in the place of their scores: parts of 8 columns each
            auto weigh = [&](auto looks, auto scaled, auto far, int c, float ratio) {
#pragma unroll
                for (int n = 0; n < KV8_TILE; n += 16) {
                    float s[16];
                    kv8m_load16(scores + (uint32_t)(c * KV8_TILE + n), s);
                    uint32_t hw[8], lw[8];
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        float w[2];
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const int at = n + j + k;
                            float x = s[j + k];
                            if (looks.value) x = at >= lo[c] && at <= hi[c] ? __uint_as_float(__float_as_uint(x) ^ sign[c]) : -INFINITY;
                            w[k] = kv8_exp2(far.value ? kv8_far_power(x, f[c], m) : fmaf(x, f[c], less));
                            total[k] += w[k];
                            if (scaled.value) w[k] *= ratio;
                        }
                        hw[j / 2] = kv8_half2(w[0], w[1]);
                        const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&hw[j / 2]));
                        lw[j / 2] = kv8_half2(w[0] - u.x, w[1] - u.y);
                    }
                    kv8m_store8(scores + (uint32_t)(c * KV8_TILE + n), hw);
                    kv8m_store8(scores + (uint32_t)(c * KV8_TILE + n + 8), lw);
                }
            };
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const float ratio = vs[c] == vt ? 1.0f : __fdiv_rn(vs[c], vt);
                if (__any_sync(0xffffffffu, fabsf(less) >= KV8_FAR))
                    weigh(std::true_type(), std::true_type(), std::true_type(), c, ratio);
                else if (!__all_sync(0xffffffffu, plain[c]))
                    weigh(std::true_type(), std::true_type(), std::false_type(), c, ratio);
                else if (!__all_sync(0xffffffffu, ratio == 1.0f))
                    weigh(std::false_type(), std::true_type(), std::false_type(), c, ratio);
                else
                    weigh(std::false_type(), std::false_type(), std::false_type(), c, ratio);
            }
            sum = fmaf(sum, shrink, total[0] + total[1]);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        ug_fence_before();
        if (half)                            // numbers in registers would take all of the barriers of an SM
            asm volatile("bar.sync 2, 128;" ::: "memory");
        else
            asm volatile("bar.sync 1, 128;" ::: "memory");
        if ((warp & 3) == 0) {
            ug_fence_after();
            const uint64_t v = kv8m_desc_values(dz_smem_addr(sm + B::WIDE + B::PANELS * B::PANEL + half * 64 * 128), B::PANEL);
            if (ug_elect()) {
#pragma unroll
                for (int part = 0; part < 2; part++)
#pragma unroll
                    for (int kk = 0; kk < 4; kk++)
                        kv8m_mma_tmem(tmem + (uint32_t)(128 + HD * half), tmem + (uint32_t)(64 * half + kk * 16 + part * 8),
                                      v + ((uint32_t)(kk * 2048) >> 4), sums_desc, part || kk ? 1u : 0u);
                ug_commit(&sums_bar[half]);
            }
            __syncwarp();
        }
        scales();                            // the next tile's, while the sums are on their way
        raw[0] = entry(i + 2, 2 * half);
        raw[1] = entry(i + 2, 2 * half + 1);
        // every warp: the widened values are free once the sums are there
        if (!dz_mbar_wait(&sums_bar[half], (uint32_t)(i & 1))) ok = false;
        ug_fence_after();
        if (busy) {
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
                int32_t raw[32];
                ug_tmem_ld32(sums + (uint32_t)c, raw);
#pragma unroll
                for (int j = 0; j < 32; j++) o[c + j] = fmaf(__int_as_float(raw[j]), vt * KV8_LOWER, o[c + j] * shrink);
            }
        }
        if (!ok) *failed = 1;
        ug_fence_before();
        __syncthreads();
        ug_fence_after();
        if (*failed) break;
    }
    if (i < mine) {                          // something did not come: the unit reads NaN, once what is under way has ended
        for (int t = i; t < mine && t < i + 3; t++) dz_mbar_wait(&codes_bar[t & 1], (uint32_t)((t >> 1) & 1));
        dz_mbar_wait(scores_bar, (uint32_t)(i & 1));
        dz_mbar_wait(&sums_bar[0], (uint32_t)(i & 1));
        dz_mbar_wait(&sums_bar[1], (uint32_t)(i & 1));
        sum = __int_as_float(0x7fc00000);
        __syncthreads();
    }
    if (warp == 0) {
        ug_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)B::COLUMNS) : "memory");
    }
    // the halves' sums, [half][pair][HD], a pair's 16-byte pieces turned by its number
    float4* join = reinterpret_cast<float4*>(sm);
#pragma unroll
    for (int c = 0; c < HD / 4; c++)
        join[(half * KV8M_PAIRS + r) * (HD / 4) + (c ^ (r & 7))] = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
    // scores that all left fp32 at -inf: no weight, but not a pair that saw nothing
    stats[half * KV8M_PAIRS + r] = make_float2(top, seen && sum == 0.0f ? 1.0f : sum);
    if (cluster > 1)
        cg::this_cluster().sync();
    else
        __syncthreads();
    // a thread has four elements of a row; several parts' loads are in flight at a time
    auto of = [&](auto* base, int part) { return cluster > 1 ? cg::this_cluster().map_shared_rank(base, part >> 1) : base; };
    auto output = [&](auto width) {
        constexpr int AT_ONCE = decltype(width)::value;
        for (int x = rank * KV8M_THREADS + (int)threadIdx.x; x < rows * (HD / 4); x += cluster * KV8M_THREADS) {
            const int row = x / (HD / 4), d = x % (HD / 4);
            float m = -INFINITY, total = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            bool any = false;
            for (int p0 = 0; p0 < 2 * cluster; p0 += AT_ONCE) {
                float2 st[AT_ONCE];
                float4 v[AT_ONCE];
#pragma unroll
                for (int p = 0; p < AT_ONCE; p++) {
                    st[p] = make_float2(-INFINITY, 0.0f);
                    v[p] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (p0 + p < 2 * cluster) {
                        const int at = (p & 1) * KV8M_PAIRS + row;
                        st[p] = of(stats, p0 + p)[at];
                        v[p] = of(join, p0 + p)[at * (HD / 4) + (d ^ (row & 7))];
                    }
                }
                float most = m;
#pragma unroll
                for (int p = 0; p < AT_ONCE; p++) most = fmaxf(most, st[p].x);
                const float f0 = m == most ? 1.0f : kv8_exp2(m - most);
                m = most;
                total *= f0;
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] *= f0;
#pragma unroll
                for (int p = 0; p < AT_ONCE; p++) {
                    const float f = st[p].x == -INFINITY ? 0.0f : st[p].x == m ? 1.0f : kv8_exp2(st[p].x - m);
                    // a part that weighs nothing may still hold a NaN, which counts; one that saw nothing is all 0
                    total = fmaf(st[p].y, f, total);
                    any |= st[p].y != 0.0f;
                    y[0] = fmaf(v[p].x, f, y[0]);
                    y[1] = fmaf(v[p].y, f, y[1]);
                    y[2] = fmaf(v[p].z, f, y[2]);
                    y[3] = fmaf(v[p].w, f, y[3]);
                }
            }
            const int pair = r0 + row;
            T* out = static_cast<T*>(a.out) + ((long long)b * a.n_tokens + pair / share) * a.ldo + (h * share + pair % share) * HD + 4 * d;
#pragma unroll
            for (int e = 0; e < 4; e++) out[e] = dz_from_float<T>(any ? y[e] / (total * KV8_LOWER) : 0.0f);
        }
    };
    if (cluster > 1)
        output(std::integral_constant<int, 8>());
    else
        output(std::integral_constant<int, 2>());
    if (cluster > 1) cg::this_cluster().sync();      // no block ends while another reads its shared memory
}

template <typename T, int HD> static cudaError_t kv8_many_t(const Kv8AttnArgs& a, long long longest, int device, cudaStream_t st) {
    static Kv8Room rooms[KV8_DEVICES];
    constexpr int smem = Kv8Many<T, HD>::SMEM;
    const auto kernel = dz_kv8_many_kernel<T, HD>;
    Kv8Room& room = rooms[device];
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(KV8M_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    if (!room.known.load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess)                // room for as many blocks as the registers hold
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
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
    const int pairs = a.n_tokens * (a.q_heads / a.c.kv_heads), blocks = (pairs + KV8M_PAIRS - 1) / KV8M_PAIRS;
    const long long units = (long long)a.c.batch * a.c.kv_heads * blocks;
    // the blocks of a cluster: the least estimated time, in tiles of a block alone on its SM (about 3 us with heads of 64). Two on
    // an SM, which the occupancy does not count for kernels with tensor memory, take 1.66 times as long, and a cluster then
    // half of the SMs; a start and an end are worth 4 tiles, a join 1 and 0.1 for each block.
    const long long visible = a.window && a.window < longest ? a.window + a.n_tokens : longest;
    const long long tiles = (visible + KV8M_KEYS - 1) / KV8M_KEYS;
    int cluster = 1;
    double best = 1e30;
    for (int c = 1; c <= KV8_CLUSTER && c <= tiles; c++) {
        const long long alone = room.clusters[c].load(std::memory_order_relaxed);
        if (alone <= 0) continue;
        const bool two = HD == 64 && units > alone;
        const long long slots = !two ? alone : c == 1 ? 2 * alone : (long long)room.clusters[(c + 1) / 2].load(std::memory_order_relaxed);
        const double each = (double)((tiles + c - 1) / c) * (two ? 1.66 : 1.0) + 4.0 + (c > 1 ? 1.0 + 0.1 * c : 0.0);
        const double t = (double)((units + slots - 1) / slots) * each;
        if (t < best) {
            best = t;
            cluster = c;
        }
    }
    cfg.gridDim = dim3((unsigned)(units * cluster));
    attr[0].val.clusterDim.x = cluster;
    cfg.attrs = cluster > 1 ? attr : attr + 1;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    CUtensorMap maps[2];
    if (!kv8_maps(a.c, HD, maps)) return cudaErrorInvalidValue;
    return cudaLaunchKernelEx(&cfg, kernel, a, maps[0], maps[1], cluster, blocks);
}

cudaError_t dz_kv8_many_launch(const Kv8AttnArgs& a, long long longest, int type, int head_dim, int device, cudaStream_t st) {
    if (type == DZ_TYPE_F32)
        return head_dim == 128 ? kv8_many_t<float, 128>(a, longest, device, st) : kv8_many_t<float, 64>(a, longest, device, st);
    if (type == DZ_TYPE_F16)
        return head_dim == 128 ? kv8_many_t<__half, 128>(a, longest, device, st) : kv8_many_t<__half, 64>(a, longest, device, st);
    return head_dim == 128 ? kv8_many_t<__nv_bfloat16, 128>(a, longest, device, st) : kv8_many_t<__nv_bfloat16, 64>(a, longest, device, st);
}

}  // namespace dz
