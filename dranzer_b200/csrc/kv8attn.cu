// Attention over the 8-bit paged caches (kv8.cuh): softmax(scale q . k) . v for
// the newest queries of every sequence, with fp32 sums and running statistics;
// of many queries in kv8many.cu.
//
// A unit is one (sequence, key head) and up to 8 NT pairs (query token, query
// head). Tokens are the rows of the MMAs of the scores, pairs their columns;
// elements of the head are the rows of the MMAs of the sums, pairs again their
// columns, so that few pairs leave few columns idle. Warps take
// tiles of 32 tokens of a unit in turn, a tile lying in one page, so that one
// scale for keys and one for values serve a whole tile. Its keys and its values
// come by TMA, each a box of 32 rows into a slot of the warp's own ring, three
// or four of them ahead (loads into registers left no room for enough of them:
// 231 us for 24 ragged sequences where the ring took 208). They
// are read as MMA operands by ldmatrix: keys as they are, values turned in units
// of two elements, so that a register holds two elements of two tokens; the
// weights turn from the scores' result into the sums' operand by movmatrix.
//
// Up to 8 pairs, keys enter the 8-bit integer MMA (m16n8k32) as their codes. A
// query is counted in steps of 2^-30 of a power of two above its largest element
// and cut into four balanced base-256 digits, so that products and sums are
// exact and nothing is widened (with keys widened a tile took 831 instructions
// where the digits took 757). With more pairs the digits' sums cost more than keys
// widened once for all of them: keys are fp16 (m16n8k16), queries fp16 too, bf16
// and fp32 ones times a power of two of their row (its largest element in [2^13,
// 2^14)), fp32 ones in two parts (22 of their 24 bits: a third part would be half
// again as many MMAs for less than the fp32 sums of the scores round). Codes
// become fp16 exactly, two at a time, by setting the exponent of 1024 above the
// byte and subtracting 1024 + 128; values always do, and weights are taken times
// 2^15 in two fp16 parts (22 bits of each; one part alone, 11 bits, would save 6%
// of a tile's instructions and show in bf16 outputs where values of both signs
// cancel). Scores of a tile take the page's key scale, the sums of a tile its
// value scale, both in fp32.
//
// Few units of long contexts go to clusters of blocks, many to a warp each
// (kv8_shape); the parts (maximum, sum of weights, sums) join at the end in
// shared memory, of a cluster through distributed shared memory.
#include <atomic>
#include <cooperative_groups.h>
#include <type_traits>

#include "dz_types.h"
#include "kv8attn.cuh"
#include "tcgen05.cuh"

namespace dz {

namespace cg = cooperative_groups;


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

template <bool FIRST>                // the first product of a sum: no registers to clear
__device__ __forceinline__ void kv8_imma(int (&d)[4], const uint32_t (&a)[4], uint2 b) {
    if (FIRST)
        asm volatile(
            "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "r"(0));
    else asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}

// Four 8 x 8 matrices of 16-bit units from shared memory, lane l giving the
// address of row l % 8 of matrix l / 8.
__device__ __forceinline__ void kv8_matrices(uint32_t (&d)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void kv8_half_matrices(uint32_t (&d)[2], uint32_t at) {       // the first two, lanes 0..15
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(d[0]), "=r"(d[1]) : "r"(at) : "memory");
}
__device__ __forceinline__ void kv8_matrices_turned(uint32_t (&d)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(at)
                 : "memory");
}

// Rows and columns of an 8 x 8 matrix of 16-bit values exchanged: lane 4 r + c held (r, 2c), (r, 2c + 1).
__device__ __forceinline__ uint32_t kv8_turn(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// A block: as many warps as the SM's registers and shared memory hold, and the
// shared memory of one: its ring, which its sums overlay at the end, its
// queries as operands, maximum, weights and whether anything was seen of each
// pair, and the ring's barriers.
template <int HD, int NT> struct Kv8Block {
    static constexpr int WARPS = HD == 64 ? (NT == 1 ? 16 : 12) : NT == 1 ? 12 : 8;
    static constexpr int SLOTS = HD == 128 && NT == 1 ? 3 : 4, SLOT = KV8_TILE * HD, PAIRS = 8 * NT;
    static constexpr int RING = SLOTS * SLOT > PAIRS * HD * 4 ? SLOTS * SLOT : PAIRS * HD * 4;
    static constexpr int QUERIES = PAIRS * HD * 4, STATS = PAIRS * 12;
    static constexpr int SMEM = 1024 + WARPS * (RING + QUERIES + STATS + SLOTS * 8);
    static_assert(SMEM <= 227 * 1024, "the shared memory of a block");
};

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(Kv8Block<HD, NT>::WARPS * 32, 1)
    dz_kv8_attn_kernel(const __grid_constant__ Kv8AttnArgs a, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, int team, int cluster, int blocks, int units) {
    using B = Kv8Block<HD, NT>;
    constexpr int PAIRS = B::PAIRS, WARPS = B::WARPS, SLOTS = B::SLOTS;
    constexpr bool DIGITS = NT == 1;
    constexpr int PARTS = std::is_same<T, float>::value ? 2 : 1;      // fp16 parts of a query's element
    constexpr int TILES = HD / 16;           // sum MMAs over a head's elements
    extern __shared__ __align__(1024) uint8_t kv8_raw[];
    uint8_t* sm = kv8_raw + ((1024u - (dz_smem_addr(kv8_raw) & 1023u)) & 1023u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float* join = reinterpret_cast<float*>(sm);                       // [warps][RING / 4]: [PAIRS][HD]
    uint2* queries = reinterpret_cast<uint2*>(sm + WARPS * B::RING);  // [warps][NT][HD / 32][4 digits][32 lanes], or
                                                                      // [warps][PARTS][NT][HD / 16][32 lanes]
    float2* stats = reinterpret_cast<float2*>(sm + WARPS * (B::RING + B::QUERIES));     // [warps][PAIRS] maximum, weights
    uint64_t* bars = reinterpret_cast<uint64_t*>(stats + WARPS * PAIRS);                // [warps][SLOTS]
    int* seens = reinterpret_cast<int*>(bars + WARPS * SLOTS);                          // [warps][PAIRS]
    uint8_t* ring = sm + warp * B::RING;
    uint64_t* bar = bars + warp * SLOTS;
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < SLOTS; i++) dz_mbar_init(&bar[i]);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int rank = cluster > 1 ? (int)(blockIdx.x % (unsigned)cluster) : 0;
    const int unit = cluster > 1 ? blockIdx.x / cluster : blockIdx.x * (WARPS / team) + warp / team;
    const int warps = team * cluster, me = cluster > 1 ? rank * WARPS + warp : warp % team;
    const int share = a.q_heads / a.c.kv_heads, pairs = a.n_tokens * share;
    int b = 0, h = 0, r0 = 0, rows = 0;
    long long first = -1;
    // entries of the table, those of the warp's next three tiles ahead: without a window they do not wait for the position
    const int shift = a.c.page == 64 ? 6 : 5;
    const int32_t* table = a.c.table;
    auto entry = [&](int i, int last) { return i <= last ? table[i >> (shift - 5)] : -1; };
    int raw[3] = {-1, -1, -1};
    if (unit < units) {
        const int blk = unit % blocks, bh = unit / blocks;
        h = bh % a.c.kv_heads;
        b = bh / a.c.kv_heads;
        r0 = blk * PAIRS;
        rows = min(PAIRS, pairs - r0);
        table += (long long)b * a.c.table_pages;
        if (!a.window) {
            const int last = (a.c.table_pages << (shift - 5)) - 1;
#pragma unroll
            for (int i = 0; i < 3; i++) raw[i] = entry(me + i * warps, last);
        }
        first = a.positions[b];
        if (kv8_skips(first)) rows = 0;
    }
    float o[TILES][NT][4];                   // elements 16 i + 2 g (0, 1) and + 1 (2, 3) of pairs 2 t, 2 t + 1
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
        const int from = low_of(0), to = min(high_of(rows - 1), (int)reach - 1);
        const int t_first = from >> 5, t_last = to < from ? -1 : to >> 5;                 // tiles
        // the warp's tiles that have a page, in turn: this one and the two after it, their entries read three ahead
        int at = t_first + me;
        if (a.window) {
#pragma unroll
            for (int i = 0; i < 3; i++) raw[i] = entry(at + i * warps, t_last);
        }
        int tile[3] = {0, 0, 0}, page[3] = {-1, -1, -1};
        auto look = [&](int which) {
            page[which] = -1;
            while (at <= t_last && page[which] < 0) {
                tile[which] = at;
                page[which] = (unsigned)raw[0] < (unsigned)a.c.pages ? raw[0] : -1;
                raw[0] = raw[1];
                raw[1] = raw[2];
                raw[2] = entry(at + 3 * warps, t_last);
                at += warps;
            }
        };
        const bool elected = ug_elect();
        unsigned flying = 0, parity = 0;     // slots that are being filled; their barriers' phases
        auto copy = [&](int slot, bool keys, int which) {
            if (page[which] < 0) return;
            if (elected) {
                dz_mbar_expect_tx(&bar[slot], B::SLOT);
                kv8_copy(ring + slot * B::SLOT, keys ? &tm_k : &tm_v,
                         h * a.c.page + (shift == 6 ? (tile[which] & 1) * KV8_TILE : 0), page[which], &bar[slot]);
            }
            flying |= 1u << slot;
        };
        auto arrived = [&](int slot) {
            const bool ok = dz_mbar_wait(&bar[slot], parity >> slot & 1u);
            parity ^= 1u << slot;
            flying &= ~(1u << slot);
            return ok;
        };
#pragma unroll
        for (int i = 0; i < 3; i++) look(i);
        copy(0, true, 0);
        copy(1, false, 0);
        copy(2, true, 1);
        if (SLOTS == 4) copy(3, false, 1);
        const float *k_scales = a.c.k_scales + h, *v_scales = a.c.v_scales + h;
        auto scale_of = [&](const float* scales) { return page[0] >= 0 ? scales[(long long)page[0] * a.c.kv_heads] : 0.0f; };
        float k_scale = scale_of(k_scales), v_scale = scale_of(v_scales) * KV8_LOWER;
        // queries as B operands, of pair 8 n + g
        uint2* qb = queries + warp * (B::QUERIES / 8) + lane;
        const bool wide = ((uintptr_t)a.q | (uintptr_t)(a.ldq * (long long)sizeof(T))) % (4 * sizeof(T)) == 0;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int r = min(r0 + 8 * n + g, pairs - 1);
            const T* q = static_cast<const T*>(a.q) + ((long long)b * a.n_tokens + r / share) * a.ldq +
                         (h * share + r % share) * HD + 4 * t;
            float x[HD / 4], peak = 0.0f;    // elements 16 c + 4 t + 0..3 for every c
            bool bad = false;
#pragma unroll
            for (int c = 0; c < HD / 16; c++) {
                T own[4];
                if (wide) {
                    if (sizeof(T) == 4)
                        *reinterpret_cast<uint4*>(own) = *reinterpret_cast<const uint4*>(q + 16 * c);
                    else
                        *reinterpret_cast<uint2*>(own) = *reinterpret_cast<const uint2*>(q + 16 * c);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) own[i] = q[16 * c + i];
                }
#pragma unroll
                for (int i = 0; i < 4; i++) x[4 * c + i] = dz_to_float(own[i]);
            }
#pragma unroll
            for (int i = 0; i < HD / 4; i++) {
                peak = fmaxf(peak, fabsf(x[i]));
                bad |= !(fabsf(x[i]) <= 3.402823466e38f);
            }
            peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
            peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
            bad |= __shfl_xor_sync(0xffffffffu, (int)bad, 1);
            bad |= __shfl_xor_sync(0xffffffffu, (int)bad, 2);
            // 2^e that takes the largest to [2^29, 2^30) or [2^13, 2^14), in two factors within fp32
            const int e = peak > 0.0f ? (DIGITS ? 29 : 13) - (int)((__float_as_uint(peak) >> 23) & 255) + 127 : 0;
            const int e0 = min(max(e, -126), 126), e1 = e - e0;
            const float up0 = __uint_as_float((unsigned)(e0 + 127) << 23), up1 = __uint_as_float((unsigned)(e1 + 127) << 23);
            float own = a.scale * 1.4426950408889634f * __uint_as_float((unsigned)(127 - e0) << 23) *
                        __uint_as_float((unsigned)(127 - e1) << 23);
            if (bad) own = __int_as_float(0x7fc00000);
            factor[n][0] = __shfl_sync(0xffffffffu, own, 8 * t);      // of pair 2 t, which lanes 8 t.. hold
            factor[n][1] = __shfl_sync(0xffffffffu, own, 8 * t + 4);
            if (DIGITS) {                    // step s: elements 32 s + 4 t + 0..3 and 16 further on
#pragma unroll
                for (int s = 0; s < HD / 32; s++) {
                    unsigned word[8];        // an element's four digits: the carries of 128 a digit, taken off again
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        word[i] = ((unsigned)(bad ? 0 : __float2int_rn(x[8 * s + i] * up0 * up1)) + 0x80808080u) ^ 0x80808080u;
                    }
#pragma unroll
                    for (int d = 0; d < 4; d++) {                // digit d of four elements side by side
                        const unsigned pick = (unsigned)(d | (d + 4) << 4);
                        uint2 v;
                        v.x = __byte_perm(__byte_perm(word[0], word[1], pick), __byte_perm(word[2], word[3], pick), 0x5410);
                        v.y = __byte_perm(__byte_perm(word[4], word[5], pick), __byte_perm(word[6], word[7], pick), 0x5410);
                        qb[((n * (HD / 32) + s) * 4 + d) * 32] = v;
                    }
                }
            } else {                         // step s: elements 16 s + 4 t + 0, 2 and + 1, 3
#pragma unroll
                for (int s = 0; s < HD / 16; s++) {
                    float v[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = x[4 * s + i] * up0 * up1;
                    const uint2 hi = make_uint2(kv8_half2(v[0], v[2]), kv8_half2(v[1], v[3]));
                    qb[(n * (HD / 16) + s) * 32] = hi;
                    if (PARTS == 2) {
                        const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&hi.x));
                        const float2 w = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
                        qb[((NT + n) * (HD / 16) + s) * 32] =
                            make_uint2(kv8_half2(v[0] - u.x, v[2] - u.y), kv8_half2(v[1] - w.x, v[3] - w.y));
                    }
                }
            }
        }
        __syncwarp();
        // the row that the lane addresses in a slot, whose 16-byte chunks are swizzled: of keys tokens 0..15 by 2 chunks, of
        // values tokens 0..31
        const int row = lane & 7, turn = HD == 128 ? row : row >> 1;
        const int k_at = (row + (lane & 8)) * HD + ((lane >> 4 ^ turn) * 16), v_at = lane * HD + turn * 16;
        bool ok = true;
        int slot = 0;
        while (page[0] >= 0) {
            const int p0 = tile[0] * KV8_TILE;
            if (!arrived(slot)) ok = false;
            const uint32_t keys = dz_smem_addr(ring + slot * B::SLOT) + k_at;
            float s[2][NT][4];               // tokens 16 i + g (0, 1) and + 8 (2, 3), pairs 2 t, 2 t + 1
            if constexpr (DIGITS) {
                int sums[2][NT][4][4];
#pragma unroll
                for (int e = 0; e < HD / 32; e++) {
                    uint32_t k[2][4];
#pragma unroll
                    for (int i = 0; i < 2; i++) kv8_matrices(k[i], (keys ^ 32 * e) + i * (16 * HD));
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int d = 0; d < 4; d++) {
                            const uint2 q = qb[((n * (HD / 32) + e) * 4 + d) * 32];
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                if (e == 0)
                                    kv8_imma<true>(sums[i][n][d], k[i], q);
                                else
                                    kv8_imma<false>(sums[i][n][d], k[i], q);
                            }
                        }
                }
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int c = 0; c < 4; c++)              // below 2^29 each
                            s[i][n][c] = fmaf((float)(sums[i][n][3][c] * 256 + sums[i][n][2][c]), 65536.0f,
                                              (float)(sums[i][n][1][c] * 256 + sums[i][n][0][c]));
            } else {
#pragma unroll
                for (int e = 0; e < HD / 16; e++) {
                    uint2 q[PARTS][NT];
#pragma unroll
                    for (int p = 0; p < PARTS; p++)
#pragma unroll
                        for (int n = 0; n < NT; n++) q[p][n] = qb[((p * NT + n) * (HD / 16) + e) * 32];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        uint32_t k[2];       // tokens 16 i + g and + 8
                        kv8_half_matrices(k, (keys ^ 16 * e) + i * (16 * HD));
                        const uint32_t ka[4] = {kv8_widen<false>(k[0]), kv8_widen<false>(k[1]), kv8_widen<true>(k[0]),
                                                kv8_widen<true>(k[1])};
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
            }
            __syncwarp();                    // the keys' slot is free: the next copy but two
            if (SLOTS == 3)
                copy(slot, false, 1);
            else
                copy(slot, true, 2);
            // scores are f times the dot products, f > 0: the products' signs turned where the scales' are not alike, and a
            // least f, so that hidden tokens stay at -inf
            if ((k_scale < 0.0f) != (a.scale < 0.0f)) {
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int c = 0; c < 4; c++) s[i][n][c] = -s[i][n][c];
            }
            float f[NT][2], vs[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    f[n][e] = fabsf(k_scale * factor[n][e]);
                    f[n][e] = f[n][e] == 0.0f ? 1.17549435e-38f : f[n][e];
                    vs[n][e] = v_scale;
                }
            if (p0 + KV8_TILE - 1 <= high_all && p0 >= low_all) {      // every pair sees the whole tile
#pragma unroll
                for (int n = 0; n < NT; n++) seen[n][0] = seen[n][1] = 1;
            } else {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
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
                        if (!any) {          // whatever the scales are
                            f[n][e] = 1.17549435e-38f;
                            vs[n][e] = 0.0f;
                        }
                        seen[n][e] |= any;
                    }
            }
            float shrink[NT][2], less[NT][2];
            bool far = false;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float m = fmaxf(fmaxf(s[0][n][e], s[0][n][2 + e]), fmaxf(s[1][n][e], s[1][n][2 + e]));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    m = fmaxf(top[n][e], m * f[n][e]);
                    shrink[n][e] = top[n][e] == m ? 1.0f : kv8_exp2(top[n][e] - m);
                    top[n][e] = m;
                    if (m == -INFINITY) m = 0.0f;
                    less[n][e] = 15.0f - m;                      // weights times 2^15
                    far |= fabsf(m) >= KV8_FAR;
                }
            auto weigh = [&](auto power) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float w = 0.0f;
#pragma unroll
                        for (int i = 0; i < 2; i++)
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                s[i][n][2 * j + e] = kv8_exp2(power(s[i][n][2 * j + e], n, e));
                                w += s[i][n][2 * j + e];
                            }
                        sum[n][e] = fmaf(sum[n][e], shrink[n][e], w);
                    }
            };
            if (__any_sync(0xffffffffu, far))
                weigh([&](float x, int n, int e) { return kv8_far_power(x, f[n][e], top[n][e]); });
            else
                weigh([&](float x, int n, int e) { return fmaf(x, f[n][e], less[n][e]); });
            // every tile: a branch for those whose maximum grew costs as many moves
#pragma unroll
            for (int i = 0; i < TILES; i++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    o[i][n][0] *= shrink[n][0];
                    o[i][n][1] *= shrink[n][1];
                    o[i][n][2] *= shrink[n][0];
                    o[i][n][3] *= shrink[n][1];
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
                        wh[i][n][j] = kv8_turn(hi);
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
                        wl[i][n][j] = kv8_turn(kv8_half2(s[i][n][2 * j] - f.x, s[i][n][2 * j + 1] - f.y));
                    }
            const int slot_v = slot + 1 == SLOTS ? 0 : slot + 1;
            if (!arrived(slot_v)) ok = false;
            if (!ok) page[1] = page[2] = -1; // nothing after this tile
            const uint32_t values = dz_smem_addr(ring + slot_v * B::SLOT) + v_at;
            {                                // this tile's scales are in use: the next one's
                const int p = page[1] >= 0 ? page[1] : page[0];
                k_scale = k_scales[(long long)p * a.c.kv_heads];
                v_scale = v_scales[(long long)p * a.c.kv_heads] * KV8_LOWER;
            }
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                uint32_t v[4];               // elements 16 i + 2 g, + 1 of tokens 8 j + 2 t, + 1
                kv8_matrices_turned(v, values ^ 16 * i);
                float part[NT][4];
#pragma unroll
                for (int st = 0; st < 2; st++) {
                    const uint32_t va[4] = {kv8_widen<false>(v[2 * st]), kv8_widen<true>(v[2 * st]),
                                            kv8_widen<false>(v[2 * st + 1]), kv8_widen<true>(v[2 * st + 1])};
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
            __syncwarp();                    // the values' slot is free
            if (SLOTS == 3)
                copy(slot_v, true, 2);
            else
                copy(slot_v, false, 2);
            tile[0] = tile[1];
            page[0] = page[1];
            tile[1] = tile[2];
            page[1] = page[2];
            if (ok)
                look(2);
            else
                page[2] = -1;
            slot = slot_v + 1 == SLOTS ? 0 : slot_v + 1;
        }
        if (!ok) {                           // a copy did not come: the unit reads NaN, once those under way have ended
            for (int i = 0; i < SLOTS; i++)
                if (flying >> i & 1u) arrived(i);
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    sum[n][e] = __int_as_float(0x7fc00000);
                    seen[n][e] = 1;
                }
        }
        __syncwarp();
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
            float* at = join + warp * (B::RING / 4) + r * HD + 2 * g;
#pragma unroll
            for (int i = 0; i < TILES; i++) *reinterpret_cast<float2*>(at + 16 * i) = make_float2(o[i][n][e], o[i][n][2 + e]);
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
#pragma unroll 4
            for (int w = 0; w < team; w++) {
                m = fmaxf(m, st[(w0 + w) * PAIRS + r].x);
                any |= sn[(w0 + w) * PAIRS + r];
            }
        }
        float total = 0.0f, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int c = 0; c < cluster; c++) {
            const float2* st = cluster > 1 ? cg::this_cluster().map_shared_rank(stats, c) : stats;
            const float* jn = cluster > 1 ? cg::this_cluster().map_shared_rank(join, c) : join;
#pragma unroll 4
            for (int w = 0; w < team; w++) {
                const int at = (w0 + w) * PAIRS + r;
                const float2 s = st[at];
                const float f = s.x == -INFINITY ? 0.0f : s.x == m ? 1.0f : kv8_exp2(s.x - m);
                // a part that weighs nothing may still hold a NaN, which counts; one that saw nothing is all 0
                const float4 v = *reinterpret_cast<const float4*>(jn + (w0 + w) * (B::RING / 4) + r * HD + d);
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
        for (int i = 0; i < 4; i++) out[i] = dz_from_float<T>(any ? y[i] / (total * KV8_LOWER) : 0.0f);
    }
    if (cluster > 1) cg::this_cluster().sync();      // no block ends while another reads its shared memory
}

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
    constexpr int PAIRS = 8 * NT, WARPS = Kv8Block<HD, NT>::WARPS, smem = Kv8Block<HD, NT>::SMEM;
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
    CUtensorMap maps[2];
    if (!kv8_maps(a.c, HD, maps)) return cudaErrorInvalidValue;
    return cudaLaunchKernelEx(&cfg, kernel, a, maps[0], maps[1], team, cluster, blocks, (int)units);
}

template <typename T>
static cudaError_t kv8_attn_h(const Kv8AttnArgs& a, long long longest, int head_dim, int device, cudaStream_t st) {
    // up to 8 pairs in 8 columns, more in 16
    const bool few = a.n_tokens * (a.q_heads / a.c.kv_heads) <= 8;
    if (head_dim == 128) return few ? kv8_attn_t<T, 128, 1>(a, longest, device, st) : kv8_attn_t<T, 128, 2>(a, longest, device, st);
    return few ? kv8_attn_t<T, 64, 1>(a, longest, device, st) : kv8_attn_t<T, 64, 2>(a, longest, device, st);
}

cudaError_t dz_kv8_attn_launch(const Kv8AttnArgs& a, long long longest, int type, int head_dim, int device, cudaStream_t st) {
    if (device < 0 || device >= KV8_DEVICES) return cudaErrorInvalidDevice;
    // pairs of a key head: 16 in a warp here, 128 in a block of kv8many.cu (8 sequences of 4000 tokens, 4 key heads, here and
    // there. Heads of 64 in fp16: 64 pairs 27 and 25 us, 80 46 and 26, 320 125 and 68; in fp32 29 and 26, 50 and 27, 137 and
    // 70. Heads of 128 in bf16: 32 pairs 28 and 38, 48 44 and 39, 128 79 and 41; in fp32 30 and 40, 49 and 41, 90 and 44)
    if (a.n_tokens * (a.q_heads / a.c.kv_heads) > (head_dim == 128 ? 32 : 64)) return dz_kv8_many_launch(a, longest, type, head_dim, device, st);
    if (type == DZ_TYPE_F32) return kv8_attn_h<float>(a, longest, head_dim, device, st);
    if (type == DZ_TYPE_F16) return kv8_attn_h<__half>(a, longest, head_dim, device, st);
    return kv8_attn_h<__nv_bfloat16>(a, longest, head_dim, device, st);
}

}  // namespace dz
