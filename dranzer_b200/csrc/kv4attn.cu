// Attention over the 4-bit ring caches (kv4.cuh), in a translation unit of its
// own.
//
// A unit is one (sequence, key head) and up to 2 NT of its (query token, query
// head) pairs. Its visible tokens go in tiles of 32 to a team of
// 1, 2, 4 or 8 warps in turn, or to the warps of a cluster of 2 to 16 blocks;
// each warp keeps its own softmax state and the states join in shared memory,
// then across the cluster. A warp's start and its part in a join cost as much
// as several tiles, so a team is no larger than it takes to fill the SMs.
//
// Products, in the 8-bit integer MMA (m16n8k32), whose sums of a tile or a
// 64-element group are exact. Codes are its A operand as they are, unsigned
// bytes holding code or 16 x code, so that one or two logic operations widen
// four of them; the 7 that a code stands above its level is taken off by the
// value that an accumulator starts at. B columns are balanced digits of base 256:
//   scores   A = 16 tokens x 32 elements of K, B = the query's digits. Its
//            elements are integers after a power of two per 64-element group.
//            Group sums times the token's scale add up in fp32.
//   values   A = 16 elements of V^T x 32 tokens, B = the digits of weight x
//            value scale (of either sign), integers after a power of two per
//            tile and group. Tile sums add up in fp32.
// A pair takes 4 of the 8 columns. Half a step is at most 2^-30 of the group's
// largest element, or of the tile's largest weight x scale: 16-bit queries are
// exact but for what lies below that. An accumulator starts at the bits of 1.5 x
// 2^23 (less the 7s): its bits read as a float are 1.5 x 2^23 plus the sum.
//
// Units of 3 or 4 pairs of 16-bit types (FV) take their values in the 16-bit MMA: weight x
// scale in two bf16 parts (2^-17 of itself), two columns for a pair, levels widened
// to bf16 and summed in the accumulators over all tiles. 2 x 8 key heads of 128, 4
// queries each, 130k tokens: 104 us, 155 with digits in two n-tiles. (Two digits
// for queries and weights of 16-bit types took 76 us, and lost small elements
// and small weights beside large ones.)
//
// Bound by instruction issue: 540 per tile of 32 tokens at head dimension 128
// and one pair, 2.5 a cycle per SM. 256 x 16 heads of 128, up to 641
// tokens: 69 us per call, 4.9 TB/s of the 6.55 that a copy reaches. With levels
// widened to fp16 pairs in m16n8k16 (two fp16 parts per fp32 weight) a tile took
// 860 instructions, most of the ALU's issue rate in widening, and the call 118
// us.
#include <cmath>

#include "kv4launch.cuh"
#include "shim.cuh"

namespace dz {

constexpr int KA_WARPS = KV4_WARPS;
constexpr int KA_TILE = KV4_TILE;
constexpr int KA_STAGES = 3;
constexpr int KA_ZERO = 0x4B400000;       // 1.5 x 2^23
constexpr float KA_ZEROF = 12582912.0f;

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

// A unsigned, B signed.
__device__ __forceinline__ void ka_mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ka_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The larger of two, NaN if either is.
__device__ __forceinline__ float ka_max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

__device__ __forceinline__ void ka_mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Levels of the nibbles at bits 0 and 16 of w as a bf16 pair: or-ed into 128,
// whose step is 1, a nibble adds itself; 135 less is the level. (lop3: both
// constants stay in registers, one instruction.)
__device__ __forceinline__ uint32_t ka_level(uint32_t w) {
    uint32_t x;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(x) : "r"(w), "r"(0x000F000Fu), "r"(0x43004300u));
    const __nv_bfloat162 y = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x),
                                     __bfloat162bfloat162(__ushort_as_bfloat16(0x4307)));
    return *reinterpret_cast<const uint32_t*>(&y);
}

// Byte d of four words (sel = d | (4 + d) << 4).
__device__ __forceinline__ uint32_t ka_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t sel) {
    return __byte_perm(__byte_perm(a, b, sel), __byte_perm(c, d, sel), 0x5410);
}

template <typename T, int HD, int NT, bool SPLIT, bool FV>
__global__ void __launch_bounds__(KA_WARPS * 32, 2) dz_kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a,
                                                                                    int team, int cluster, int pair_blocks,
                                                                                    int units) {
    using C = KaCfg<HD>;
    constexpr int CPP = 4;                   // columns of a pair
    // Pairs of an n-tile; lane t has columns of pair 2 t / CPP. SPLIT: where they
    // would fill half the columns at most, the two value groups take a half
    // each: columns 0..3 of the weights' digits belong to group 0, 4..7 to
    // group 1, and a lane weighs the values of its columns' group alone (256 x
    // 16 units of 640 tokens, one pair each: 69 us instead of 76).
    constexpr int PPT = (SPLIT ? 4 : 8) / CPP;
    constexpr int PAIRS = NT * PPT;          // pairs of a block
    constexpr int GR = C::GROUPS, GA = SPLIT ? 1 : GR;   // value groups of a lane's columns
    static_assert(!SPLIT || (NT == 1 && GR == 2), "two groups share one n-tile");
    // FV: values in the 16-bit MMA, one n-tile for 4 pairs. The scores' two n-tiles
    // hold pairs 2 c and 2 c + 1 in column block c, so that lane t ends up with
    // pair t alone: one softmax state a lane.
    static_assert(!FV || (NT == 2 && !SPLIT), "the four lanes of a row have a pair each");
    constexpr int SN = FV ? 1 : NT;          // softmax states of a lane
    extern __shared__ __align__(16) uint8_t smem[];
    asm volatile("griddepcontrol.wait;" ::: "memory");   // launched while the kernel before ends
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % cluster, tw = warp % team;      // the warp's place in its team
    int unit = blockIdx.x / cluster * (KA_WARPS / team) + warp / team;
    if (unit >= units) return;               // whole teams of a single block
    const int pb = unit % pair_blocks;
    unit /= pair_blocks;
    const int hk = unit % a.c.kv_heads, b = unit / a.c.kv_heads;
    const long long first = a.positions[b] + a.pos_add;
    if (kv4_skips(first)) return;   // the whole team, or cluster, leaves
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
        const int s0 = slot_of(v0);
        // whole, neither across the sinks' end nor round the ring: one run of slots
        const bool run = v0 + KA_TILE <= count && (v0 >= nsink || v0 + KA_TILE <= nsink) && s0 + KA_TILE <= cap;
        const int r = lane / CH, c = lane % CH;
        const uint32_t d = s + r * C::ROW + (HD == 128 ? (c ^ (r & 2)) : c) * 16;   // (r + 8 i) & 2 == r & 2
        const uint32_t ds = s + 2 * C::CODES + lane * GR * 4;
        if (run) {
            const uint8_t* k = kc + (long long)s0 * C::ROW + lane * 16;
            const uint8_t* v = vc + (long long)s0 * C::ROW + lane * 16;
#pragma unroll
            for (int i = 0; i < KA_TILE / RPI; i++) {
                ka_copy16(d + i * 512, k + i * 512, true);
                ka_copy16(d + C::CODES + i * 512, v + i * 512, true);
            }
            ka_copy_small<GR * 4>(ds, ksc + ((long long)s0 + lane) * GR, true);
            ka_copy_small<GR * 4>(ds + C::SCALES, vsc + ((long long)s0 + lane) * GR, true);
            return;
        }
#pragma unroll
        for (int i = 0; i < KA_TILE / RPI; i++) {
            const int v = v0 + r + i * RPI;
            const long long off = (long long)(v < count ? slot_of(v) : 0) * C::ROW + c * 16;
            ka_copy16(d + i * 512, kc + off, v < count);
            ka_copy16(d + C::CODES + i * 512, vc + off, v < count);
        }
        const bool valid = v0 + lane < count;
        const long long off = (long long)(valid ? slot_of(v0 + lane) : 0) * GR;
        ka_copy_small<GR * 4>(ds, ksc + off, valid);
        ka_copy_small<GR * 4>(ds + C::SCALES, vsc + off, valid);
    };

    const int ntiles = (count + KA_TILE - 1) / KA_TILE, step = team * cluster;
    const int tile0 = rank * team + tw;
#pragma unroll
    for (int i = 0; i < KA_STAGES - 1; i++) {
        if (tile0 + i * step < ntiles) issue(tile0 + i * step, i);
        ka_commit();
    }

    // ---- query digits: column g of n-tile n is digit g % CPP of pair pair0 +
    // n PPT + g / CPP; lane t has elements 16 t .. 16 t + 15 of each group, the
    // even ones in B step 0, the odd ones in step 1, as the codes' nibbles fall
    const uint32_t dsel = (uint32_t)(g % CPP) * 0x11u + 0x40u;          // digit d: d | (4 + d) << 4
    uint32_t qd[NT][GR][2][2];
    int zero[NT][GR][2];                     // where the accumulators of columns 2t, 2t + 1 start
    float qw[NT][GR][2];                     // and what their sums count: 256^digit / the group's power / 16
    bool qbad[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int pair = pair0 + (FV ? 2 * (g / CPP) + n : n * PPT + (SPLIT ? g % 4 : g) / CPP);
        const bool live = pair < pairs;
        const T* q = static_cast<const T*>(a.q) +
                     ((long long)b * a.n_tokens + (live ? pair / share : 0)) * a.ldq +
                     (long long)(hk * share + (live ? pair % share : 0)) * HD + 16 * t;
        bool bad = false;
#pragma unroll
        for (int gr = 0; gr < GR; gr++) {
            float x[16], top = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                x[i] = live ? dz_to_float(q[64 * gr + i]) : 0.0f;
                top = fmaxf(top, fabsf(x[i]));
                bad |= !(fabsf(x[i]) <= 3.402823466e38f);
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // the power of two that puts the largest in [2^29, 2^30)
            const int e = min(127 + 29 - (int)(__float_as_uint(top) >> 23), 126);
            const float f = __int_as_float((127 + e) << 23);
            uint32_t y[16];
#pragma unroll
            for (int i = 0; i < 16; i++) y[i] = (uint32_t)__float2int_rn(x[i] * f) + 0x808080u;
            const uint32_t flip = g % CPP < 3 ? 0x80808080u : 0u;   // the lower digits' 128 taken off
            int sum = 0;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint32_t* z = y + 8 * j + h;
                    qd[n][gr][h][j] = ka_bytes(z[0], z[2], z[4], z[6], dsel) ^ flip;
                    sum = __dp4a((int)qd[n][gr][h][j], 0x01010101, sum);
                }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const int start0 = KA_ZERO - 112 * sum;
            const float digit = g % CPP == 0 ? 0.0625f : g % CPP == 1 ? 16.0f : g % CPP == 2 ? 4096.0f : 1048576.0f;
            const float weight = digit * __int_as_float((127 - e) << 23);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                zero[n][gr][i] = __shfl_sync(0xffffffffu, start0, 8 * t + 4 * i);
                qw[n][gr][i] = __shfl_sync(0xffffffffu, weight, 8 * t + 4 * i);
            }
        }
        qbad[n] = __any_sync(0xfu << (lane & 28), bad);
    }
    const int tp = SPLIT ? 2 * t % 4 : 2 * t;    // the lane's first column, as pairs count them
    auto lane_pair = [&](int n) { return FV ? t : n * PPT + tp / CPP; };   // of the block's
    // ---- the score factor and the visible range of the lane's pairs
    float sfac[SN];                          // scale x log2 e (NaN for a query that holds one)
    int see_sink[SN], see_hi[SN], see_lo[SN];
    const bool masked = a.n_tokens > 1;
#pragma unroll
    for (int n = 0; n < SN; n++) {
        // (columns 2t of the n-tile are lane 8 t's; of FV's pair t, n-tile t % 2's block t / 2, lane 16 (t / 2)'s)
        bool bad = __shfl_sync(0xffffffffu, qbad[n], FV ? 16 * (t >> 1) : 8 * t);
        if constexpr (FV) {
            const bool odd = __shfl_sync(0xffffffffu, qbad[1], 16 * (t >> 1));
            bad = t & 1 ? odd : bad;
        }
        sfac[n] = bad ? __int_as_float(0x7fc00000) : a.scale * 1.4426950408889634f;
        const int pair = min(pair0 + lane_pair(n), pairs - 1);
        const long long pos = first + pair / share;
        see_sink[n] = (int)min(pos, (long long)INT32_MAX);
        see_hi[n] = (int)max(-1LL, pos - lo);
        see_lo[n] = a.window ? (int)max(-1LL, pos - a.window - lo) : -1;
    }

    // tiles of later positions that every pair of the block sees: rel in (all_lo, all_hi]
    const int all_hi = (int)max(-1LL, first + j_lo - lo);
    const int all_lo = a.window ? (int)max(-1LL, first + j_hi - a.window - lo) : -1;

    float m[SN], l[SN];
    // elements 64 gr + 8 g + 2 k (and 16 x that of + 1), the lane's digits; FV: two parts of each of the two
    constexpr int AW = FV ? 4 : 2;
    float acc[SN][GA * 4][AW];
#pragma unroll
    for (int n = 0; n < SN; n++) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < GA * 4; i++)
#pragma unroll
            for (int j = 0; j < AW; j++) acc[n][i][j] = 0.0f;
    }
    // the weights' digits as C columns 2t and 2t + 1 count them
    const float wd0 = t & 1 ? 65536.0f : 1.0f, wd1 = t & 1 ? 16777216.0f : 256.0f;
    const uint32_t wflip = g % CPP < 3 ? 0x80808080u : 0u;

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
        constexpr uint32_t HIGH = 0xF0F0F0F0u, LOW = 0x0F0F0F0Fu;

        // scores of tokens g, g + 8, g + 16, g + 24
        float x[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int r = 0; r < 4; r++) x[n][r] = 0.0f;
#pragma unroll
        for (int blk = 0; blk < 2; blk++) {
            const int r0 = blk * 16 + g, r1 = r0 + 8;
#pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                // 8 bytes at 8 t of the group's 32: rows r0 and r1 (r1 & 2 == r0 & 2)
                const int at = HD == 128 ? ((2 * gr + (t >> 1)) ^ (g & 2)) * 16 + 8 * (t & 1) : 8 * t;
                const uint2 w0 = *reinterpret_cast<const uint2*>(st + r0 * C::ROW + at);
                const uint2 w1 = *reinterpret_cast<const uint2*>(st + r1 * C::ROW + at);
                const float k0 = ks[r0 * GR + gr], k1 = ks[r1 * GR + gr];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    int c[4] = {zero[n][gr][0], zero[n][gr][1], zero[n][gr][0], zero[n][gr][1]};
                    ka_mma(c, (w0.x << 4) & HIGH, (w1.x << 4) & HIGH, (w0.y << 4) & HIGH, (w1.y << 4) & HIGH,
                             qd[n][gr][0][0], qd[n][gr][0][1]);
                    ka_mma(c, w0.x & HIGH, w1.x & HIGH, w0.y & HIGH, w1.y & HIGH, qd[n][gr][1][0], qd[n][gr][1][1]);
                    const float u0 = qw[n][gr][0], u1 = qw[n][gr][1];
                    const float s0 = fmaf(__int_as_float(c[1]) - KA_ZEROF, u1, (__int_as_float(c[0]) - KA_ZEROF) * u0);
                    const float s1 = fmaf(__int_as_float(c[3]) - KA_ZEROF, u1, (__int_as_float(c[2]) - KA_ZEROF) * u0);
                    x[n][2 * blk] = fmaf(s0, k0, x[n][2 * blk]);
                    x[n][2 * blk + 1] = fmaf(s1, k1, x[n][2 * blk + 1]);
                }
            }
        }
        const int v0 = tile * KA_TILE;
        const int rel0 = v0 - nsink;
        const bool edge = v0 + KA_TILE > count ||
                          (masked && !(rel0 > all_lo && v0 >= nsink && rel0 + KA_TILE - 1 <= all_hi));
        uint32_t bw[SN][GA][2];              // digits of weight x value scale (of either sign)
        uint32_t wb[GA][4];                  // FV: a part of them, tokens t + 8 i and t + 8 i + 4
        float back[SN][GA][2];               // what columns 2t, 2t + 1 count
        if constexpr (FV) {
            // even lanes have digits 0 and 1 of both n-tiles' pairs, odd ones 2 and 3: even take the first n-tile's others
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float other = __shfl_xor_sync(0xffffffffu, t & 1 ? x[0][r] : x[1][r], 1);
                x[0][r] = (t & 1 ? x[1][r] : x[0][r]) + other;
            }
        }
#pragma unroll
        for (int n = 0; n < SN; n++) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                if constexpr (!FV) x[n][r] += __shfl_xor_sync(0xffffffffu, x[n][r], 1);   // the pair's other digits
                x[n][r] *= sfac[n];
            }
            unsigned hidden = 0;
            if (edge) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int v = v0 + r * 8 + g, rel = v - nsink;
                    const bool see = v < nsink ? v <= see_sink[n] : rel <= see_hi[n] && rel > see_lo[n];
                    if (!see || v >= count) {
                        x[n][r] = -INFINITY;
                        hidden |= 1u << r;
                    }
                }
            }
            float top = fmaxf(fmaxf(x[n][0], x[n][1]), fmaxf(x[n][2], x[n][3]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            if (__any_sync(0xffffffffu, top > m[n])) {
                const float mn = fmaxf(m[n], top);
                const float c = m[n] == -INFINITY ? 0.0f : ka_exp2(m[n] - mn);   // nothing was summed before
                l[n] *= c;
                m[n] = mn;
#pragma unroll
                for (int i = 0; i < GA * 4; i++)
#pragma unroll
                    for (int j = 0; j < AW; j++) acc[n][i][j] *= c;
            }
            const float ref = m[n] == -INFINITY ? 0.0f : m[n];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[n][r] = ka_exp2(x[n][r] - ref);
                l[n] += x[n][r];
            }
            // another query's token may hold a NaN scale: its weight is marked by its sign, and makes no product
            // (a token that is seen and whose weight is 0 makes one: its NaN counts)
            if (masked && edge) {
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (hidden >> r & 1) x[n][r] = -0.0f;
            }
            // the weights in B layout: tokens t + 4 i, column g
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; i++)
                p[i] = __shfl_sync(0xffffffffu, x[n][i >> 1], (t + 4 * (i & 1)) * 4 + g / 2);
#pragma unroll
            for (int gr = 0; gr < GA; gr++) {
                float w[8], wtop = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) w[i] = p[i] * vs[(t + 4 * i) * GR + (SPLIT ? g >> 2 : gr)];
                if (masked && edge) {
#pragma unroll
                    for (int i = 0; i < 8; i++) w[i] = __float_as_uint(p[i]) == 0x80000000u ? 0.0f : w[i];
                }
                if constexpr (FV) {          // column g is part g % 2 of pair g / 2: the weight in bf16, or what is left of it
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(w[i], w[i + 1]);
                        const uint32_t hi = *reinterpret_cast<const uint32_t*>(&h);
                        const __nv_bfloat162 r = __floats2bfloat162_rn(w[i] - __uint_as_float(hi << 16),
                                                                       w[i + 1] - __uint_as_float(hi & 0xffff0000u));
                        wb[gr][i / 2] = g & 1 ? *reinterpret_cast<const uint32_t*>(&r) : hi;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) wtop = ka_max_nan(wtop, fabsf(w[i]));
                    wtop = ka_max_nan(wtop, __shfl_xor_sync(0xffffffffu, wtop, 1));
                    wtop = ka_max_nan(wtop, __shfl_xor_sync(0xffffffffu, wtop, 2));
                    // the power of two that puts the largest in [2^29, 2^30); 0x808080 added, the lower bytes less
                    // 128 are the lower digits, the last byte the top one. Below 2^-97 the weights fade out.
                    constexpr uint32_t TOP = 29;
                    const uint32_t e = max(__float_as_uint(wtop) & 0x7F800000u, 30u << 23);
                    const float f = __uint_as_float(((254u + TOP) << 23) - e);
                    uint32_t y[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) y[i] = (uint32_t)__float2int_rn(w[i] * f) + 0x808080u;
                    bw[n][gr][0] = ka_bytes(y[0], y[1], y[2], y[3], dsel) ^ wflip;
                    bw[n][gr][1] = ka_bytes(y[4], y[5], y[6], y[7], dsel) ^ wflip;
                    // its inverse, NaN where a weight is not finite
                    const float inv = fmaf(wtop, 0.0f, __uint_as_float(e - (TOP << 23)));
                    back[n][gr][0] = __shfl_sync(0xffffffffu, inv, 8 * t) * wd0;
                    back[n][gr][1] = __shfl_sync(0xffffffffu, inv, 8 * t + 4) * wd1;
                }
            }
        }
        // ---- values
        auto codes = [&](int gr, uint32_t (&w)[8]) {     // word g of the group's eight, tokens t + 4 i
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int r = t + 4 * i;
                const int at = HD == 128 ? ((2 * gr + (g >> 2)) ^ (t & 2)) * 16 + 4 * (g & 3) : 4 * g;
                w[i] = *reinterpret_cast<const uint32_t*>(st + C::CODES + r * C::ROW + at);
            }
        };
        if constexpr (FV) {
            // rows g and g + 8 of an A operand are elements 8 g + 2 byte and + 1, its columns tokens t + 16 s + 4 i
#pragma unroll
            for (int gr = 0; gr < GR; gr++) {
                uint32_t w[8];
                codes(gr, w);
#pragma unroll
                for (int byte = 0; byte < 4; byte++) {
                    const uint32_t sel = (uint32_t)byte * 0x11u | (uint32_t)(4 + byte) * 0x1100u;
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const uint32_t u = __byte_perm(w[4 * s], w[4 * s + 1], sel);
                        const uint32_t v = __byte_perm(w[4 * s + 2], w[4 * s + 3], sel);
                        ka_mma_bf16(acc[0][4 * gr + byte], ka_level(u), ka_level(u >> 4), ka_level(v), ka_level(v >> 4),
                                    wb[gr][2 * s], wb[gr][2 * s + 1]);
                    }
                }
            }
        } else {
            int start[SN][GA][4];
#pragma unroll
            for (int n = 0; n < SN; n++)
#pragma unroll
                for (int gr = 0; gr < GA; gr++) {
                    int c[4] = {0, 0, 0, 0};     // the digits' sums over the tile
                    ka_mma(c, 0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u, bw[n][gr][0], bw[n][gr][1]);
                    start[n][gr][0] = KA_ZERO - 7 * c[0];
                    start[n][gr][1] = KA_ZERO - 7 * c[1];
                    start[n][gr][2] = KA_ZERO - 112 * c[0];
                    start[n][gr][3] = KA_ZERO - 112 * c[1];
                }
            // Byte `byte` of the tokens: element 8 g + 2 byte in the low halves, the next one in the high halves.
            auto multiply = [&](const uint32_t (&w)[8], int byte, int n, int gr, int (&c)[4]) {
                const uint32_t sel = (uint32_t)byte * 0x11u + 0x40u;
                const uint32_t b0 = ka_bytes(w[0], w[1], w[2], w[3], sel), b1 = ka_bytes(w[4], w[5], w[6], w[7], sel);
#pragma unroll
                for (int i = 0; i < 4; i++) c[i] = start[n][gr][i];
                ka_mma(c, b0 & LOW, b0 & HIGH, b1 & LOW, b1 & HIGH, bw[n][gr][0], bw[n][gr][1]);
            };
            auto add = [&](const int (&c)[4], int n, int gr, int byte) {
                float* o = acc[n][4 * gr + byte];
                o[0] = fmaf(__int_as_float(c[0]) - KA_ZEROF, back[n][gr][0], o[0]);
                o[0] = fmaf(__int_as_float(c[1]) - KA_ZEROF, back[n][gr][1], o[0]);
                o[1] = fmaf(__int_as_float(c[2]) - KA_ZEROF, back[n][gr][0], o[1]);
                o[1] = fmaf(__int_as_float(c[3]) - KA_ZEROF, back[n][gr][1], o[1]);
            };
            if constexpr (SPLIT) {
                uint32_t w0[8], w1[8];
                codes(0, w0);
                codes(1, w1);
#pragma unroll
                for (int byte = 0; byte < 4; byte++) {
                    int c0[4], c1[4];
                    multiply(w0, byte, 0, 0, c0);
                    multiply(w1, byte, 0, 0, c1);
#pragma unroll
                    for (int i = 0; i < 4; i++) c0[i] = t < 2 ? c0[i] : c1[i];   // the lane's columns' group
                    add(c0, 0, 0, byte);
                }
            } else {
#pragma unroll
                for (int gr = 0; gr < GR; gr++) {
                    uint32_t w[8];
                    codes(gr, w);
#pragma unroll
                    for (int byte = 0; byte < 4; byte++)
#pragma unroll
                        for (int n = 0; n < SN; n++) {
                            int c[4];
                            multiply(w, byte, n, gr, c);
                            add(c, n, gr, byte);
                        }
                }
            }
        }
    }

    // ---- the warp's sums in units of its 2^m: lane (g, t) has elements 64 gr + 8 g .. + 7 of
    // pair tp / CPP (SPLIT: of group t / 2 alone)
    ka_wait<0>();
    __syncwarp();
#pragma unroll
    for (int n = 0; n < SN; n++) {
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], 4);
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], 8);
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], 16);
#pragma unroll
        for (int k = 0; k < GA * 4; k++) {
            if constexpr (FV) {
                acc[n][k][0] += acc[n][k][1];
                acc[n][k][1] = acc[n][k][2] + acc[n][k][3];
            } else {
                acc[n][k][0] += __shfl_xor_sync(0xffffffffu, acc[n][k][0], 1);
                acc[n][k][1] += __shfl_xor_sync(0xffffffffu, acc[n][k][1], 1);
                acc[n][k][1] *= 0.0625f;
            }
        }
    }
    auto store_out = [&](int p, int d, float v) {
        static_cast<T*>(a.out)[((long long)b * a.n_tokens + p / share) * a.ldo +
                               (long long)(hk * share + p % share) * HD + d] = dz_from_float<T>(v);
    };
    const bool speaks = FV || !(t & 1);        // of two lanes with the same sums
    const int e0 = (SPLIT ? 64 * (t >> 1) : 0) + 8 * g;
    if (team * cluster == 1) {
#pragma unroll
        for (int n = 0; n < SN; n++) {
            const int p = pair0 + lane_pair(n);
            if (p >= pairs || !speaks) continue;
            T* o = static_cast<T*>(a.out) + ((long long)b * a.n_tokens + p / share) * a.ldo +
                   (long long)(hk * share + p % share) * HD + e0;
            const float inv = 1.0f / l[n];
#pragma unroll
            for (int gr = 0; gr < GA; gr++)
#pragma unroll
                for (int k = 0; k < 8; k++) o[64 * gr + k] = dz_from_float<T>(acc[n][4 * gr + k / 2][k % 2] * inv);
        }
        return;
    }

    // ---- join: each warp's sums, m and l over its ring; [pair][OS]
    constexpr int OS = HD + 16;              // float4 stores of 2 g and 4 t meet a bank twice at most
    constexpr int MINE = KA_STAGES * C::STAGE / 4;
    static_assert(PAIRS * OS + 2 * PAIRS <= MINE, "a warp's part of the join lies over its ring");
    float* so = reinterpret_cast<float*>(my);
#pragma unroll
    for (int n = 0; n < SN; n++) {
        const int pair = lane_pair(n);
        if (!speaks) continue;
#pragma unroll
        for (int gr = 0; gr < GA; gr++)
#pragma unroll
            for (int k = 0; k < 4; k += 2)
                *reinterpret_cast<float4*>(so + pair * OS + 64 * gr + e0 + 2 * k) =
                    make_float4(acc[n][4 * gr + k][0], acc[n][4 * gr + k][1], acc[n][4 * gr + k + 1][0],
                                acc[n][4 * gr + k + 1][1]);
        if (g == 0 && (!SPLIT || t < 2)) {
            so[PAIRS * OS + pair] = m[n];
            so[PAIRS * OS + PAIRS + pair] = l[n];
        }
    }
    // the team's barrier (teams of one block have barriers of their own: their lengths differ)
    asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / team), "r"(team * 32) : "memory");
    const float* t0 = reinterpret_cast<const float*>(smem) + (warp - tw) * MINE;
    float* co = reinterpret_cast<float*>(smem + C::RING);       // a cluster's block: [pair][HD], [pair], [pair]
    for (int i = tw * 32 + lane; i < PAIRS * HD; i += team * 32) {
        const int pair = i / HD, d = i % HD, p = pair0 + pair;
        if (p >= pairs) break;
        float mx = -INFINITY;
        for (int w = 0; w < team; w++) mx = fmaxf(mx, t0[w * MINE + PAIRS * OS + pair]);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        float o = 0.0f, s = 0.0f;
        for (int w = 0; w < team; w++) {
            const float* q = t0 + w * MINE;
            const float f = ka_exp2(q[PAIRS * OS + pair] - ref);
            o = fmaf(q[pair * OS + d], f, o);
            s = fmaf(q[PAIRS * OS + PAIRS + pair], f, s);
        }
        if (cluster == 1) {
            store_out(p, d, o / s);
        } else {
            co[i] = o;
            if (d == 0) {
                co[PAIRS * HD + pair] = mx;
                co[PAIRS * HD + PAIRS + pair] = s;
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
        store_out(p, i % HD, o / s);
    }
    // no block leaves while another may still read its shared memory
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}

// Pairs of a block.
template <int NT, bool SPLIT> constexpr int ka_pairs() { return NT * 2 / (SPLIT ? 2 : 1); }

template <int HD, int NT, bool SPLIT> constexpr int ka_smem() {
    constexpr int pairs = ka_pairs<NT, SPLIT>();
    return KaCfg<HD>::RING + (pairs * HD + 2 * pairs) * 4;
}

template <typename T, int HD, int NT, bool SPLIT, bool FV>
static cudaError_t ka_launch(const Kv4AttnArgs& a, int device, cudaStream_t st) {
    static Kv4Room rooms[KV4_DEVICES];
    return kv4_launch(dz_kv4_attn_kernel<T, HD, NT, SPLIT, FV>, rooms, a, ka_pairs<NT, SPLIT>(), ka_smem<HD, NT, SPLIT>(), device,
                      st);
}

// One n-tile where it holds all pairs of a key head, else two (more leave one
// block to an SM).
template <typename T, int HD> static cudaError_t ka_launch_n(const Kv4AttnArgs& a, int device, cudaStream_t st) {
    const int pairs = a.n_tokens * (a.q_heads / a.c.kv_heads);
    if constexpr (HD == 128)
        if (pairs <= ka_pairs<1, true>()) return ka_launch<T, HD, 1, true, false>(a, device, st);
    if (pairs <= ka_pairs<1, false>()) return ka_launch<T, HD, 1, false, false>(a, device, st);
    return ka_launch<T, HD, 2, false, sizeof(T) == 2>(a, device, st);
}

// Pairs of a key head up to which tokens are the MMA's rows; above, pairs are
// (kv4chunk.cu). Both on 8 x 4 key heads of 128 that see 4160 tokens, fp32: 4
// pairs 22 us each, 8 pairs 27 against 24; fp16: 4 pairs 18 against 17, 8 pairs 21
// against 19 (2 x 8 key heads, 130k tokens, bf16: 4 pairs 104 against 165, 8 pairs 155
// against 167), 16 pairs 30 against 22. Of 64, fp32: 8 pairs 16 against 19, 16 pairs
// 23 against 21; fp16: 8 pairs 13 against 15, 16 pairs 18 against 17.
static int ka_limit(int head_dim) { return head_dim == 128 ? 4 : 8; }

template <typename T> static cudaError_t ka_launch_t(const Kv4AttnArgs& a, int head_dim, int device, cudaStream_t st) {
    return head_dim == 128 ? ka_launch_n<T, 128>(a, device, st) : ka_launch_n<T, 64>(a, device, st);
}

cudaError_t dz_kv4_attn_launch(const Kv4AttnArgs& a, int type, int head_dim, int device, cudaStream_t st) {
    if ((long long)a.n_tokens * (a.q_heads / a.c.kv_heads) > ka_limit(head_dim))
        return dz_kv4_chunk_launch(a, type, head_dim, device, st);
    if (type == DZ_TYPE_F32) return ka_launch_t<float>(a, head_dim, device, st);
    if (type == DZ_TYPE_F16) return ka_launch_t<__half>(a, head_dim, device, st);
    return ka_launch_t<__nv_bfloat16>(a, head_dim, device, st);
}

}  // namespace dz
