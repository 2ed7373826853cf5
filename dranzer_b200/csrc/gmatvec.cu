// Group-scaled 4-bit products: the device layout, the kernel (gmatvec.cuh) and
// the C entry points, in a translation unit of their own.
#include "dz_cuda.h"

#include <atomic>
#include <cmath>
#include <new>
#include <type_traits>

#include "gmatvec.cuh"
#include "shim.cuh"

namespace dz {

__device__ __forceinline__ int gmv_code(const uint8_t* packed, long long i) {
    return (packed[i >> 1] >> ((i & 1) * 4)) & 15;
}

// Where element (k, n) of a record lies: its word, the bit of its nibble.
__device__ __forceinline__ int gmv_word(int kk, int c) {
    return (kk >> 5) * 128 + ((c & 7) * 4 + ((kk >> 3) & 3)) * 4 + (c >> 3);
}
__device__ __forceinline__ int gmv_bit(int kk) { return (kk & 4) ? 8 * (kk & 3) : 8 * (kk & 3) + 4; }

// One thread per word of the records' codes. `bad` is set for a code of 15.
__global__ void dz_gmv_repack_kernel(const uint8_t* __restrict__ packed, GmvMatrix w, int* __restrict__ bad) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (long long)w.ntiles * w.nblocks * (GMV_CODES / 4)) return;
    const int word = (int)(i % (GMV_CODES / 4));
    const long long r = i / (GMV_CODES / 4);
    const int piece = word >> 7, lane = (word >> 2) & 31, q = word & 3;
    const int n = (int)(r / w.nblocks) * GMV_TILE + (lane >> 2) + 8 * q;
    const int k0 = (int)(r % w.nblocks) * GMV_BLOCK + 32 * piece + 8 * (lane & 3);
    uint32_t v = 0;
    if (n < w.N) {
        for (int k = k0; k < min(k0 + 8, w.K); k++) {
            const int c = gmv_code(packed, (long long)k * w.N + n);
            if (c > 14) *bad = 1;
            v |= ((uint32_t)(c - 7) & 15u) << gmv_bit(k);
        }
    }
    *reinterpret_cast<uint32_t*>(w.rec + r * w.rec_bytes + 4 * word) = v;
}

// One thread per scale slot of the records. `bad` is set for a scale that is
// negative or not finite.
template <typename S>
__global__ void dz_gmv_scales_kernel(const S* __restrict__ scales, GmvMatrix w, int* __restrict__ bad) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int per = GMV_BLOCK / w.group * GMV_TILE;
    if (i >= (long long)w.ntiles * w.nblocks * per) return;
    const int at = (int)(i % per);
    const long long r = i / per;
    const int n = (int)(r / w.nblocks) * GMV_TILE + at % GMV_TILE;
    const int k = (int)(r % w.nblocks) * GMV_BLOCK + at / GMV_TILE * w.group;
    S s = dz_from_float<S>(0.0f);
    if (n < w.N && k < w.K) {
        s = scales[(long long)(k / w.group) * w.N + n];
        const float f = dz_to_float(s);
        if (!(f >= 0.0f && f <= 3.402823466e38f)) *bad = 2;
    }
    reinterpret_cast<S*>(w.rec + r * w.rec_bytes + GMV_CODES)[at] = s;
}

// One thread per element: dst = scale * level.
template <typename S> __global__ void dz_gmv_dequant_kernel(GmvMatrix w, float* __restrict__ dst) {
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (long long)w.K * w.N) return;
    const int k = (int)(i / w.N), n = (int)(i % w.N);
    const uint8_t* rec = w.rec + ((long long)(n / GMV_TILE) * w.nblocks + k / GMV_BLOCK) * w.rec_bytes;
    const int kk = k % GMV_BLOCK, c = n % GMV_TILE;
    const uint32_t word = reinterpret_cast<const uint32_t*>(rec)[gmv_word(kk, c)];
    const int level = (int)(word << (28 - gmv_bit(kk))) >> 28;
    dst[i] = dz_to_float(reinterpret_cast<const S*>(rec + GMV_CODES)[kk / w.group * GMV_TILE + c]) * (float)level;
}

// ------------------------------------------------------------------ product
//
// Every activation keeps its own precision, whatever stands beside it, in one of
// two forms; sums are fp32 from a scale group on.
//
// Several rows: the 16-bit MMA (m16n8k16) with fp32 sums, whose products are
// exact. Levels -7..7 are exact in fp16 and bf16, fp16 and bf16 activations enter
// as they are, and an fp32 one as three bf16 parts of eight bits each, a column
// of B each (P m + p is part p of row m). Widening costs most of the
// instructions: a nibble xor-ed into the low mantissa bits of 1032 (fp16; the next
// nibble too, as 16 times it) or of 136 / 1024 (bf16, whose step there is 1 / 1024)
// adds it, one subtraction (or fma) leaves the level.
//
// One row: the 8-bit integer MMA (m16n8k32), which takes a quarter of that
// widening. The block's 128 activations are scaled by a power of two that puts
// the largest in [2^21, 2^22) and cut into 8 balanced base-256 digits, one for
// each column of B: three of the integer part, three of the next 23 bits, two
// of the next 15. What lies 2^-60 below the largest is lost. Digit sums over a
// scale group are exact (16 x 7 x 128 x 128 < 2^22): an accumulator starts at the
// bits of 1.5 x 2^23, whose step is 1, so that its bits read as a float are
// 1.5 x 2^23 plus the sum. Times scale and digit weight they add up in fp32.
//
// Work. A cluster of 1 to 8 blocks (16 for the longest rows) takes a contiguous range of tiles; its
// blocks take a share of the rows of W each (so that each stages only its
// share of the activations), and a block's eight warps equal contiguous
// ranges of its (tile, block) records, whatever tile borders lie inside. A
// warp streams its records through its own ring of cp.async stages and meets
// no barrier before the end: the warp that has a tile's first record keeps its
// sum in the tile's place, a warp that continues a tile keeps it in its own.
// Then the parts add up in a fixed order, over warps, then over the cluster.
//
// On one B200, per call: 1 x 4096 x 32000 (fp32, fp16 scales) 14.5 us, 4.7 TB/s, bound by
// HBM while records stream; 1 x 2048 x 2048 3.4 us, the latency of its phases; 8 x
// 2048 x 8192 (bf16) 6.0 us and 16 x 4099 x 5003 (fp16, groups of 32) 12.8 us, staging
// and widening. One row through the 16-bit MMA took 17.1 us for the first. With
// digits for all rows (three of fp32, two of 16 bits, against a block's largest
// element) they took 14.0, 3.2, 7.7 and 16.4 us, and lost the small elements beside
// large ones. The one-thread-per-column form took 157 us for the first; a barrier
// per tile 20 us; a cluster barrier per tile 29 us.

constexpr int GMV_DEVICES = 64;         // devices whose launch state is kept
constexpr int GMV_ZERO = 0x4B400000;    // 1.5 x 2^23
constexpr float GMV_ZEROF = 12582912.0f;

__device__ __forceinline__ void gmv_mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ void gmv_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void gmv_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// (w & mask) ^ base in one instruction: both constants stay in registers.
__device__ __forceinline__ uint32_t gmv_mask_xor(uint32_t w, uint32_t mask, uint32_t base) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(y) : "r"(w), "r"(mask), "r"(base));
    return y;
}

// Levels of a word's rows 0, 2 (first) and 1, 3 (second) for i = 0, of rows 4, 6
// and 5, 7 for i = 1, as pairs of the MMA's type. A nibble is the level's two's
// complement: its top bit flipped, it is the level + 8.
__device__ __forceinline__ uint32_t gmv_level_low(uint32_t w) {
    const uint32_t x = gmv_mask_xor(w, 0x000F000Fu, 0x64086408u);
    const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x6408)));   // 1032
    return *reinterpret_cast<const uint32_t*>(&a);
}
__device__ __forceinline__ uint32_t gmv_level_high(uint32_t w) {
    const uint32_t x = gmv_mask_xor(w, 0x00F000F0u, 0x64806480u);
    const __half2 a = __hfma2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(0x2C00)),    // 1/16
                              __half2half2(__ushort_as_half(0xD480)));                                          // -72
    return *reinterpret_cast<const uint32_t*>(&a);
}
__device__ __forceinline__ uint32_t gmv_level_bf16(uint32_t w) {   // level / 1024
    const uint32_t x = gmv_mask_xor(w, 0x000F000Fu, 0x3E083E08u);
    const __nv_bfloat162 a = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x),
                                     __bfloat162bfloat162(__ushort_as_bfloat16(0x3E08)));                  // 136 / 1024
    return *reinterpret_cast<const uint32_t*>(&a);
}
__device__ __forceinline__ void gmv_levels(uint32_t w, int i, uint32_t& first, uint32_t& second, __half) {
    first = i ? gmv_level_low(w) : gmv_level_high(w);
    second = i ? gmv_level_low(w >> 8) : gmv_level_high(w >> 8);
}
__device__ __forceinline__ void gmv_levels(uint32_t w, int i, uint32_t& first, uint32_t& second, __nv_bfloat16) {
    first = gmv_level_bf16(i ? w : w >> 4);
    second = gmv_level_bf16(i ? w >> 8 : w >> 12);
}

// What an activation type takes in the MMA, and in how many columns of a row.
// UNIT: what a result's sums are counted in. bf16 levels are a 1024th, so that a
// group's sum (at most 7 x 128 of its largest activation) stays in fp32's range
// before its scale takes it back (results below 2^-116 lose bits to it).
template <typename T> struct GmvType {
    using Mma = T;
    static constexpr int PARTS = 1;
    static constexpr float UNIT = std::is_same<T, __half>::value ? 1.0f : 1024.0f;
};
template <> struct GmvType<float> {
    using Mma = __nv_bfloat16;
    static constexpr int PARTS = 3;
    static constexpr float UNIT = 1024.0f;
};

// E consecutive activations (16 bytes: 4 fp32 or 8 of 16 bits) from element k
// of a row of K, zero past the end. wide: rows start on 16-byte boundaries.
template <int E> __device__ __forceinline__ uint4 gmv_load(const void* x, long long row, int k, int K, bool wide) {
    uint4 q;
    if (E == 4) {
        const uint32_t* p = static_cast<const uint32_t*>(x) + row + k;
        if (wide && k + E <= K) return *reinterpret_cast<const uint4*>(p);
        q.x = k < K ? p[0] : 0u;
        q.y = k + 1 < K ? p[1] : 0u;
        q.z = k + 2 < K ? p[2] : 0u;
        q.w = k + 3 < K ? p[3] : 0u;
        return q;
    }
    const uint16_t* p = static_cast<const uint16_t*>(x) + row + k;
    if (wide && k + E <= K) return *reinterpret_cast<const uint4*>(p);
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = k + i < K ? p[i] : 0u;
    q.x = h[0] | h[1] << 16;
    q.y = h[2] | h[3] << 16;
    q.z = h[4] | h[5] << 16;
    q.w = h[6] | h[7] << 16;
    return q;
}

// Stages 16 bytes of a row's activations in its columns, `stride` bytes apart,
// eight elements in the order 0 2 1 3 4 6 5 7 of gmv_levels. x + 0 x turns an
// infinity into a NaN, so that the whole row reads NaN also where its level is
// not 0 (as fp32's parts do: infinity less infinity).
template <typename T2> __device__ __forceinline__ void gmv_stage16(uint8_t* to, const uint4& q, T2 zero) {
    uint32_t w[4] = {__byte_perm(q.x, q.y, 0x5410), __byte_perm(q.x, q.y, 0x7632), __byte_perm(q.z, q.w, 0x5410),
                     __byte_perm(q.z, q.w, 0x7632)};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const T2 v = *reinterpret_cast<const T2*>(&w[i]), r = __hfma2(v, zero, v);
        w[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
    *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void gmv_stage(uint8_t* to, int, const uint4& q, __half) {
    gmv_stage16(to, q, __half2half2(__ushort_as_half(0)));
}
__device__ __forceinline__ void gmv_stage(uint8_t* to, int, const uint4& q, __nv_bfloat16) {
    gmv_stage16(to, q, __bfloat162bfloat162(__ushort_as_bfloat16(0)));
}
// An fp32 value is the sum of the upper halves of x, of what is left of it and of
// what is left then: eight of its 24 bits each, without a rounding (but for bits
// below 2^-133).
__device__ __forceinline__ void gmv_stage(uint8_t* to, int stride, const uint4& q, float) {
    float r[4] = {__uint_as_float(q.x), __uint_as_float(q.y), __uint_as_float(q.z), __uint_as_float(q.w)};
#pragma unroll
    for (int p = 0; p < 3; p++) {
        uint2 w;
        w.x = __byte_perm(__float_as_uint(r[0]), __float_as_uint(r[2]), 0x7632);
        w.y = __byte_perm(__float_as_uint(r[1]), __float_as_uint(r[3]), 0x7632);
        *reinterpret_cast<uint2*>(to + p * stride) = w;
#pragma unroll
        for (int i = 0; i < 4; i++) r[i] -= __uint_as_float(__float_as_uint(r[i]) & 0xffff0000u);
    }
}

// Digits of four consecutive activations, `stride` bytes apart; f is the block's power of two.
__device__ __forceinline__ void gmv_stage_digits(uint8_t* to, int stride, const float (&v)[4], float f) {
    uint32_t y[3][4];         // an integer's digits in its low bytes, those below the top one + 128
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float a = fmaf(v[i], f, GMV_ZEROF), r = fmaf(v[i], f, GMV_ZEROF - a);
        const float b = fmaf(r, 8388608.0f, GMV_ZEROF), u = fmaf(r, 8388608.0f, GMV_ZEROF - b);
        const float c = fmaf(u, 32768.0f, GMV_ZEROF);
        // 0x40 of byte 2 belongs to 1.5 x 2^23: 0xC0 more takes it out
        y[0][i] = __float_as_uint(a) + 0x00C08080u;
        y[1][i] = __float_as_uint(b) + 0x00C08080u;
        y[2][i] = __float_as_uint(c) + 0x80u;
    }
#pragma unroll
    for (int d = 0; d < GMV_DIGITS; d++) {
        const uint32_t(&z)[4] = y[d / 3], sel = (uint32_t)(d % 3) | (uint32_t)(4 + d % 3) << 4;
        const uint32_t flip = d % 3 == 2 || d == 7 ? 0u : 0x80808080u;
        *reinterpret_cast<uint32_t*>(to + d * stride) =
            __byte_perm(__byte_perm(z[0], z[1], sel), __byte_perm(z[2], z[3], sel), 0x5410) ^ flip;
    }
}
// What digit d counts in units of the block's power: 2^-4 for the levels' factor 16 taken back.
__device__ __forceinline__ float gmv_digit_weight(int d) {
    const int e = d < 3 ? 8 * d - 4 : d < 6 ? 8 * (d - 3) - 27 : 8 * (d - 6) - 42;
    return __int_as_float((127 + e) << 23);
}

// Where share i of n things among `of` begins: shares differ by at most one.
__device__ __forceinline__ int gmv_share(unsigned n, unsigned i, unsigned of) {
    const unsigned q = n / of, r = n - q * of;
    return (int)(q * i + r * i / of);
}

template <int GPB, typename S, typename T, int NT>   // scale groups of a block, scale and activation type, column tiles of 8
__global__ void __launch_bounds__(GMV_WARPS * 32, gmv_blocks(NT, GPB)) dz_gmv_kernel(
    const __grid_constant__ GmvArgs a, const __grid_constant__ GmvPlan plan) {
    using Mma = typename GmvType<T>::Mma;
    constexpr int P = GmvType<T>::PARTS, E = 16 / (int)sizeof(T), COLS = NT ? NT : 1;
    using L = GmvSmem<P, NT>;
    constexpr int REC = GMV_CODES + GPB * GMV_TILE * (int)sizeof(S), CHUNKS = REC / 16;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int head_tile[GMV_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % plan.cluster, who = blockIdx.x / plan.cluster;
    const int M = plan.rows, stride = L::stride(plan.slice);
    uint8_t* columns = smem + L::ring(REC);
    float* fx = reinterpret_cast<float*>(columns + GMV_DIGITS * stride);       // digits' weights [record of the slice][digit]
    float* mine = reinterpret_cast<float*>(columns + L::columns(M, plan.slice)) + warp * L::TILE;
    float* parts = mine + (GMV_WARPS - warp) * L::TILE;                        // [tile][M][32]
    float* heads = parts + plan.tiles * GMV_TILE * M;                          // [warp][M][32]

    // (32-bit divisions only: a 64-bit one costs some hundred cycles before the first load)
    const unsigned nblocks = a.w.nblocks;
    const int kb0 = (int)(nblocks * rank / (unsigned)plan.cluster);
    const int nb = (int)(nblocks * (rank + 1) / (unsigned)plan.cluster) - kb0;   // >= 1: cluster <= nblocks
    const int tile0 = (int)(gmv_share(a.w.ntiles, who, plan.clusters));
    const int nt = gmv_share(a.w.ntiles, who + 1, plan.clusters) - tile0;

    // ---- this warp's records: numbers r0..r1-1 of the block's nt x nb, tile major
    const unsigned all = (unsigned)nt * nb;
    const int r0 = gmv_share(all, warp, GMV_WARPS), r1 = gmv_share(all, warp + 1, GMV_WARPS);
    const long long tile_bytes = (long long)a.w.nblocks * REC, skip = tile_bytes - (long long)nb * REC;
    int ti = r0 / nb, kb = r0 - ti * nb;                                       // the consumer's place
    const uint8_t* src = a.w.rec + (tile0 + ti) * tile_bytes + (long long)(kb0 + kb) * REC + lane * 16;
    int pk = kb, left = r1 - r0;                                               // the producer's
    uint8_t* my = smem + warp * GMV_STAGES * REC;
    const uint32_t my_s = (uint32_t)__cvta_generic_to_shared(my) + lane * 16;
    int pstage = 0;
    auto produce = [&] {
        if (left > 0) {
            left--;
            const uint32_t dst = my_s + pstage * REC;
#pragma unroll
            for (int c = 0; c < CHUNKS; c += 32)
                if (c + 32 <= CHUNKS || lane < CHUNKS - c)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + c * 16), "l"(src + c * 16));
            src += REC;
            if (++pk == nb) {
                pk = 0;
                src += skip;
            }
        }
        asm volatile("cp.async.commit_group;");
        pstage = pstage + 1 == GMV_STAGES ? 0 : pstage + 1;
    };
    produce();
    // The weights are nobody's output; activations and y wait for the kernel
    // before. (Letting the next kernel start before this one ends: 13.2 against
    // 13.9 us back to back in a graph for 1 x 4096 x 32000, but 17.4 against 13.7
    // when calls are issued one by one about as fast as they run.)
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // ---- activations to columns, 16 bytes at a time; the first four loads of a
    // thread go out ahead of the rest of the ring (behind it they would wait for
    // the weights), four more while the last are worked on
    constexpr int AHEAD = 4, THREADS = GMV_WARPS * 32, PER = GMV_BLOCK / E;   // chunks of a block
    const bool wide = (((uintptr_t)a.x | (uintptr_t)(a.ldx * (int)sizeof(T))) & 15) == 0;
    const int per = nb * PER;                          // of a row
    int m = 0, c = threadIdx.x;
    while (c >= per) { c -= per; m++; }
    uint4 raw[2][AHEAD];
    int at[2][AHEAD];                                  // row and chunk; -1: none
    auto fetch = [&](uint4 (&r)[AHEAD], int (&to)[AHEAD]) {
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            to[u] = -1;
            if (m < M) {
                to[u] = NT ? P * m * stride + c * E * 2 : c;
                r[u] = gmv_load<E>(a.x, (long long)m * a.ldx, kb0 * GMV_BLOCK + c * E, a.w.K, wide);
                c += THREADS;
                while (c >= per) { c -= per; m++; }
            }
        }
    };
    auto work = [&](const uint4 (&r)[AHEAD], const int (&to)[AHEAD]) {
        if constexpr (NT > 0) {
#pragma unroll
            for (int u = 0; u < AHEAD; u++)
                if (to[u] >= 0) gmv_stage(columns + to[u], stride, r[u], T());
        } else {
            // a block's chunks lie in neighbouring lanes of one warp, all of them there or none
            unsigned top[AHEAD];             // bits of the largest magnitude: above 0x7f7fffff it is not finite
            float v[AHEAD][E];
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                const uint32_t q[4] = {r[u].x, r[u].y, r[u].z, r[u].w};
                top[u] = 0;
#pragma unroll
                for (int j = 0; j < E; j++) {
                    if (E == 4) v[u][j] = __uint_as_float(q[j % 4]);
                    else if (std::is_same<T, __half>::value)
                        v[u][j] = __half2float(__ushort_as_half((unsigned short)(q[j / 2 % 4] >> 16 * (j & 1))));
                    else v[u][j] = __uint_as_float(j & 1 ? q[j / 2 % 4] & 0xffff0000u : q[j / 2 % 4] << 16);
                    top[u] = max(top[u], __float_as_uint(v[u][j]) & 0x7fffffffu);
                }
                if (to[u] < 0) top[u] = 0;
                top[u] = __reduce_max_sync(PER == 32 ? 0xffffffffu : lane < 16 ? 0xffffu : 0xffff0000u, top[u]);
            }
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                if (to[u] < 0) continue;
                // the power stays a normal float; of a block below 2^-86, digits that count less than 2^-149 are lost
                const int s = min(127 + 21 - (int)(top[u] >> 23), 126);
                const float f = __int_as_float((127 + s) << 23);
#pragma unroll
                for (int j = 0; j < E; j += 4) {
                    const float z[4] = {v[u][j], v[u][j + 1], v[u][j + 2], v[u][j + 3]};
                    gmv_stage_digits(columns + to[u] * E + j, stride, z, f);
                }
                const int d = to[u] % PER;
                if (d < GMV_DIGITS)
                    fx[to[u] / PER * GMV_DIGITS + d] = top[u] > 0x7f7fffffu ? __int_as_float(0x7fc00000)
                                                                           : __int_as_float((127 - s) << 23) * gmv_digit_weight(d);
            }
        }
    };
    fetch(raw[0], at[0]);
#pragma unroll
    for (int i = 0; i < GMV_STAGES - 2; i++) produce();
    while (__any_sync(0xffffffffu, at[0][0] >= 0)) {
        fetch(raw[1], at[1]);
        work(raw[0], at[0]);
        if (!__any_sync(0xffffffffu, at[1][0] >= 0)) break;
        fetch(raw[0], at[0]);
        work(raw[1], at[1]);
    }
    __syncthreads();

    // ---- records
    const uint8_t* col[COLS]; // this lane's columns (those past P M read the last one; nobody reads their sums)
#pragma unroll
    for (int n = 0; n < COLS; n++)
        col[n] = NT ? columns + min(n * 8 + g, P * M - 1) * stride + 16 * t : columns + g * stride + 8 * t;
    float out[COLS][8];       // columns g, g + 8 (0..3), g + 16, g + 24 (4..7) of W by columns 2t, 2t + 1 of B
#pragma unroll
    for (int n = 0; n < COLS; n++)
#pragma unroll
        for (int r = 0; r < 8; r++) out[n][r] = 0.0f;
    bool head = kb != 0 && r0 < r1;   // the first tile is another warp's to begin
    if (lane == 0) head_tile[warp] = head ? ti : -1;
    int cstage = 0;
    for (int r = r0; r < r1; r++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(GMV_STAGES - 2));
        __syncwarp();
        produce();
        const uint8_t* st = my + cstage * REC;
        cstage = cstage + 1 == GMV_STAGES ? 0 : cstage + 1;
        const S* scale = reinterpret_cast<const S*>(st + GMV_CODES) + g;
        float part[8];
#pragma unroll
        for (int gi = 0; gi < GPB; gi++) {
            float s[4];
#pragma unroll
            for (int q = 0; q < 4; q++) s[q] = dz_to_float(scale[gi * GMV_TILE + 8 * q]);
            if constexpr (NT == 0) {
                int acc[2][4];
#pragma unroll
                for (int q = 0; q < 8; q++) acc[q >> 2][q & 3] = GMV_ZERO;
#pragma unroll
                for (int k = gi * (4 / GPB); k < (gi + 1) * (4 / GPB); k++) {   // 32 rows each
                    const uint4 w = *reinterpret_cast<const uint4*>(st + k * 512 + lane * 16);
                    const uint2 b = *reinterpret_cast<const uint2*>(col[0] + kb * GMV_BLOCK + k * 32);
                    constexpr uint32_t HIGH = 0xF0F0F0F0u;
                    gmv_mma(acc[0], w.x & HIGH, w.y & HIGH, (w.x << 4) & HIGH, (w.y << 4) & HIGH, b);
                    gmv_mma(acc[1], w.z & HIGH, w.w & HIGH, (w.z << 4) & HIGH, (w.w << 4) & HIGH, b);
                }
#pragma unroll
                for (int q = 0; q < 8; q++) {
                    const float v = __int_as_float(acc[q >> 2][q & 3]) - GMV_ZEROF;
                    part[q] = gi ? fmaf(v, s[q >> 1], part[q]) : v * s[q >> 1];
                }
            } else {
                float acc[COLS][2][4];
#pragma unroll
                for (int n = 0; n < COLS; n++)
#pragma unroll
                    for (int q = 0; q < 8; q++) acc[n][q >> 2][q & 3] = 0.0f;
#pragma unroll
                for (int k = gi * (4 / GPB); k < (gi + 1) * (4 / GPB); k++) {
                    const uint4 w = *reinterpret_cast<const uint4*>(st + k * 512 + lane * 16);
                    uint4 b[COLS];
#pragma unroll
                    for (int n = 0; n < COLS; n++)
                        b[n] = *reinterpret_cast<const uint4*>(col[n] + (kb * GMV_BLOCK + k * 32) * 2);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        uint32_t f0[4], f1[4];   // columns g, g + 8; g + 16, g + 24
                        gmv_levels(w.x, i, f0[0], f0[2], Mma());
                        gmv_levels(w.y, i, f0[1], f0[3], Mma());
                        gmv_levels(w.z, i, f1[0], f1[2], Mma());
                        gmv_levels(w.w, i, f1[1], f1[3], Mma());
#pragma unroll
                        for (int n = 0; n < COLS; n++) {
                            const uint32_t b0 = i ? b[n].z : b[n].x, b1 = i ? b[n].w : b[n].y;
                            gmv_mma(acc[n][0], f0, b0, b1, Mma());
                            gmv_mma(acc[n][1], f1, b0, b1, Mma());
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < COLS; n++)
#pragma unroll
                    for (int q = 0; q < 8; q++) out[n][q] = fmaf(acc[n][q >> 2][q & 3], s[q >> 1], out[n][q]);
            }
        }
        if constexpr (NT == 0) {
            const float2 f = *reinterpret_cast<const float2*>(fx + kb * GMV_DIGITS + 2 * t);
#pragma unroll
            for (int q = 0; q < 8; q++) out[0][q] = fmaf(part[q], q & 1 ? f.y : f.x, out[0][q]);
        }
        if (++kb < nb && r + 1 < r1) continue;
        // the tile ends, or the warp's range does: add a row's parts or digits, the smallest first, keep the sum
#pragma unroll
        for (int n = 0; n < COLS; n++)
#pragma unroll
            for (int q = 0; q < 8; q++) {
                mine[(g + 8 * (q >> 1)) * L::LD + 8 * n + 2 * t + (q & 1)] = out[n][q];
                out[n][q] = 0.0f;
            }
        __syncwarp();
        float* to = head ? heads + warp * GMV_TILE * M : parts + ti * GMV_TILE * M;
#pragma unroll 4
        for (int m = 0; m < M; m++) {
            const float* p = mine + lane * L::LD + P * m;
            if (NT == 0)
                to[lane] = ((((p[6] + p[7]) + p[3]) + p[4]) + p[5]) + ((p[0] + p[1]) + p[2]);
            else
                to[m * GMV_TILE + lane] = P == 3 ? (p[2] + p[1]) + p[0] : p[0];
        }
        __syncwarp();
        head = false;
        kb = 0;
        ti++;
    }
    asm volatile("cp.async.wait_group 0;");
    __syncthreads();

    // ---- the block's parts in one place: warps that continue a tile, in order
    for (int o = threadIdx.x; o < GMV_TILE * M; o += GMV_WARPS * 32)
#pragma unroll
        for (int w = 1; w < GMV_WARPS; w++)
            if (head_tile[w] >= 0) parts[head_tile[w] * GMV_TILE * M + o] += heads[w * GMV_TILE * M + o];
    if (plan.cluster == 1) {
        __syncthreads();
    } else {
        asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    }
    const uint32_t parts_s = (uint32_t)__cvta_generic_to_shared(parts);
    for (int i = rank * GMV_WARPS * 32 + threadIdx.x; i < nt * GMV_TILE * M; i += plan.cluster * GMV_WARPS * 32) {
        const int tile = i / (GMV_TILE * M), m = i / GMV_TILE % M, n = (tile0 + tile) * GMV_TILE + i % GMV_TILE;
        float s = 0.0f;
        if (plan.cluster == 1) {
            s = parts[i];
        } else {
            for (int c = 0; c < plan.cluster; c++) {
                uint32_t at;
                float v;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(parts_s + 4 * i), "r"(c));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
                s += v;
            }
        }
        if (n < a.w.N) static_cast<T*>(a.y)[(long long)m * a.ldy + n] = dz_from_float<T>(NT ? s * GmvType<T>::UNIT : s);
    }
    // no block leaves while another may still read its shared memory
    if (plan.cluster > 1) asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}

template <int GPB, typename S, typename T, int NT>
static cudaError_t gmv_launch_t(const GmvArgs& a, const GmvPlan& plan, int device, cudaStream_t st) {
    auto* k = dz_gmv_kernel<GPB, S, T, NT>;
    static std::atomic<bool> ready[GMV_DEVICES];
    if (device >= GMV_DEVICES || !ready[device].load(std::memory_order_relaxed)) {
        cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, GMV_SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        if (device < GMV_DEVICES) ready[device].store(true, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(plan.clusters * plan.cluster));
    cfg.blockDim = dim3(GMV_WARPS * 32);
    cfg.dynamicSmemBytes = (size_t)GmvSmem<GmvType<T>::PARTS, NT>::total(a.w.rec_bytes, plan);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = plan.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = plan.cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, a, plan);
}

template <int GPB, typename S>
static cudaError_t gmv_launch_n(const GmvArgs& a, const GmvPlan& plan, int device, cudaStream_t st) {
    const int n = gmv_col_tiles(a.type == DZ_TYPE_F32 ? GmvType<float>::PARTS : 1, plan.rows);
    if (plan.digits)
        return a.type == DZ_TYPE_F32   ? gmv_launch_t<GPB, S, float, 0>(a, plan, device, st)
               : a.type == DZ_TYPE_F16 ? gmv_launch_t<GPB, S, __half, 0>(a, plan, device, st)
                                       : gmv_launch_t<GPB, S, __nv_bfloat16, 0>(a, plan, device, st);
    if (a.type == DZ_TYPE_F32)
        return n == 1   ? gmv_launch_t<GPB, S, float, 1>(a, plan, device, st)
               : n == 2 ? gmv_launch_t<GPB, S, float, 2>(a, plan, device, st)
               : n == 3 ? gmv_launch_t<GPB, S, float, 3>(a, plan, device, st)
                        : gmv_launch_t<GPB, S, float, 6>(a, plan, device, st);
    if (a.type == DZ_TYPE_F16)
        return n == 1 ? gmv_launch_t<GPB, S, __half, 1>(a, plan, device, st) : gmv_launch_t<GPB, S, __half, 2>(a, plan, device, st);
    return n == 1 ? gmv_launch_t<GPB, S, __nv_bfloat16, 1>(a, plan, device, st)
                  : gmv_launch_t<GPB, S, __nv_bfloat16, 2>(a, plan, device, st);
}

static cudaError_t gmv_room(int device, const GmvRoom** out) {
    static GmvRoom rooms[GMV_DEVICES];
    if (device < 0 || device >= GMV_DEVICES) return cudaErrorInvalidDevice;
    GmvRoom& r = rooms[device];
    if (!r.known.load(std::memory_order_acquire)) {
        auto* k = dz_gmv_kernel<1, float, float, 0>;
        cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, GMV_SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        for (int two = 0; two < 2 && e == cudaSuccess; two++)
            for (int c = 0; c < 5 && e == cudaSuccess; c++) {
                cudaLaunchConfig_t cfg = {};
                cfg.gridDim = dim3(16);
                cfg.blockDim = dim3(GMV_WARPS * 32);
                cfg.dynamicSmemBytes = two ? GMV_SMEM2 : GMV_SMEM;
                cudaLaunchAttribute attr[1];
                attr[0].id = cudaLaunchAttributeClusterDimension;
                attr[0].val.clusterDim.x = 1u << c;
                attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
                cfg.attrs = attr;
                cfg.numAttrs = 1;
                int n = 0;
                e = cudaOccupancyMaxActiveClusters(&n, k, &cfg);
                r.clusters[two][c].store(n, std::memory_order_relaxed);
            }
        if (e != cudaSuccess) return e;
        r.known.store(true, std::memory_order_release);
    }
    *out = &r;
    return cudaSuccess;
}

static GmvShape gmv_shape(const GmvMatrix& w, int type) {
    return GmvShape{w.ntiles, w.nblocks, w.group, w.rec_bytes, type == DZ_TYPE_F32 ? GmvType<float>::PARTS : 1};
}

cudaError_t dz_gmv_launch(const GmvArgs& a, int device, cudaStream_t st) {
    const GmvRoom* room;
    const cudaError_t err = gmv_room(device, &room);
    if (err != cudaSuccess) return err;
    GmvArgs b = a;
    GmvPlan plan;
    const GmvShape shape = gmv_shape(a.w, a.type);
    const int bytes = (int)type_bytes(a.type);
    for (int tile = 0, tiles; tile < a.w.ntiles; tile += tiles) {   // all of them at once but for the widest matrices
        tiles = gmv_plan_tiles(shape, a.w.ntiles - tile, a.M, *room, &plan);
        if (!tiles) return cudaErrorNotSupported;
        b.w.rec = a.w.rec + (long long)tile * a.w.nblocks * a.w.rec_bytes;
        b.w.ntiles = tiles;
        b.w.N = a.w.N - tile * GMV_TILE;
        for (int m = 0; m < a.M; m += plan.rows) {
            if (m && !gmv_plan(gmv_shape(b.w, a.type), a.M - m, *room, &plan)) return cudaErrorNotSupported;
            b.x = static_cast<const uint8_t*>(a.x) + (long long)m * a.ldx * bytes;
            b.y = static_cast<uint8_t*>(a.y) + ((long long)m * a.ldy + (long long)tile * GMV_TILE) * bytes;
            cudaError_t e;
            if (a.w.group == 128)
                e = a.w.scale_f16 ? gmv_launch_n<1, __half>(b, plan, device, st) : gmv_launch_n<1, float>(b, plan, device, st);
            else if (a.w.group == 64)
                e = a.w.scale_f16 ? gmv_launch_n<2, __half>(b, plan, device, st) : gmv_launch_n<2, float>(b, plan, device, st);
            else
                e = a.w.scale_f16 ? gmv_launch_n<4, __half>(b, plan, device, st) : gmv_launch_n<4, float>(b, plan, device, st);
            if (e != cudaSuccess) return e;
        }
    }
    return cudaSuccess;
}

}  // namespace dz

using namespace dz;

struct dz_cuda_gmatrix {
    int device;
    GmvMatrix m;
};

// K and N up to 2^24 and at most 2^30 records keep the kernels' indexes in range.
constexpr size_t GMV_MAX_DIM = (size_t)1 << 24;

static int gmv_check(const dz_grouped_blob_t* w) {
    if (!w || !w->packed || !w->scales) return fail(DZ_E_INVALID, "gmatrix: null argument");
    if (w->rows == 0 || w->cols == 0 || w->rows > GMV_MAX_DIM || w->cols > GMV_MAX_DIM)
        return fail(DZ_E_INVALID, "gmatrix: rows and cols must be 1..%zu", GMV_MAX_DIM);
    if (w->group != 32 && w->group != 64 && w->group != 128)
        return fail(DZ_E_INVALID, "gmatrix: groups hold 32, 64 or 128 rows, not %zu", w->group);
    if (w->scale_type != DZ_TYPE_F32 && w->scale_type != DZ_TYPE_F16)
        return fail(DZ_E_INVALID, "gmatrix: scales are fp32 or fp16");
    if (w->packed_size != (w->rows * w->cols + 1) / 2 || w->scale_count != ((w->rows - 1) / w->group + 1) * w->cols)
        return fail(DZ_E_INVALID, "gmatrix: %zu code bytes and %zu scales do not fit %zu x %zu in groups of %zu",
                    w->packed_size, w->scale_count, w->rows, w->cols, w->group);
    return DZ_OK;
}

// A failed call's status; its error is not left for a later call to find.
static int gmv_fail(const char* what, cudaError_t e) {
    (void)cudaGetLastError();
    return fail(e == cudaErrorMemoryAllocation ? DZ_E_NOMEM : DZ_E_DEVICE, "%s: %s", what, cudaGetErrorString(e));
}

// Lays w out into m->rec on `device`, the current one; the staging copies live here.
static int gmv_fill(const dz_grouped_blob_t* w, GmvMatrix* m, int device, cudaStream_t st, uint8_t** codes,
                    uint8_t** scales, int** bad) {
    const size_t sb = w->scale_count * (m->scale_f16 ? 2 : 4);
    const long long recs = (long long)m->ntiles * m->nblocks;
    DZ_CUDA(cudaMalloc(&m->rec, (size_t)recs * m->rec_bytes));
    DZ_CUDA(cudaMalloc(codes, w->packed_size));
    DZ_CUDA(cudaMalloc(scales, sb));
    DZ_CUDA(cudaMalloc(bad, 4));
    // sources in device memory may still be written by any stream of theirs
    bool waited = false;
    for (const void* src : {(const void*)w->packed, w->scales}) {
        cudaPointerAttributes at;
        if (cudaPointerGetAttributes(&at, src) != cudaSuccess) {
            (void)cudaGetLastError();
            continue;
        }
        if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) continue;
        if (!waited) DZ_CUDA(cudaDeviceSynchronize());
        waited = true;
        if (at.device != device) {
            DeviceGuard other(at.device);
            if (!other.ok) return fail(DZ_E_DEVICE, "cannot select device %d", at.device);
            DZ_CUDA(cudaDeviceSynchronize());
        }
    }
    DZ_CUDA(cudaMemcpyAsync(*codes, w->packed, w->packed_size, cudaMemcpyDefault, st));
    DZ_CUDA(cudaMemcpyAsync(*scales, w->scales, sb, cudaMemcpyDefault, st));
    DZ_CUDA(cudaMemsetAsync(*bad, 0, 4, st));
    const long long words = recs * (GMV_CODES / 4), slots = recs * (GMV_BLOCK / m->group * GMV_TILE);
    dz_gmv_repack_kernel<<<(unsigned)((words + 255) / 256), 256, 0, st>>>(*codes, *m, *bad);
    if (m->scale_f16)
        dz_gmv_scales_kernel<<<(unsigned)((slots + 255) / 256), 256, 0, st>>>((const __half*)*scales, *m, *bad);
    else
        dz_gmv_scales_kernel<<<(unsigned)((slots + 255) / 256), 256, 0, st>>>((const float*)*scales, *m, *bad);
    DZ_CUDA(cudaGetLastError());
    int why = 0;
    DZ_CUDA(cudaMemcpyAsync(&why, *bad, 4, cudaMemcpyDeviceToHost, st));
    DZ_CUDA(cudaStreamSynchronize(st));
    if (why) return fail(DZ_E_INVALID, why == 1 ? "gmatrix: a code of 15" : "gmatrix: a negative or non-finite scale");
    return DZ_OK;
}

extern "C" int dz_cuda_gmatrix_create(int device, const dz_grouped_blob_t* w, dz_cuda_gmatrix_t** out) {
    if (!out) return fail(DZ_E_INVALID, "null output handle");
    *out = nullptr;
    int rc = gmv_check(w);
    if (rc) return rc;
    DeviceGuard g(device);
    if (!g.ok) return fail(DZ_E_DEVICE, "cannot select device %d", device);
    GmvMatrix m;
    m.K = (int)w->rows;
    m.N = (int)w->cols;
    m.group = (int)w->group;
    m.scale_f16 = w->scale_type == DZ_TYPE_F16;
    m.ntiles = (m.N + GMV_TILE - 1) / GMV_TILE;
    m.nblocks = (m.K + GMV_BLOCK - 1) / GMV_BLOCK;
    m.rec_bytes = GMV_CODES + GMV_BLOCK / m.group * GMV_TILE * (m.scale_f16 ? 2 : 4);
    GmvPlan plan;
    const GmvRoom* room;
    DZ_CUDA(gmv_room(device, &room));
    if ((long long)m.ntiles * m.nblocks > (1LL << 30)) return fail(DZ_E_UNSUPPORTED, "gmatrix: too many weights");
    if (!gmv_plan_tiles(gmv_shape(m, DZ_TYPE_F32), 1, 1, *room, &plan))
        return fail(DZ_E_UNSUPPORTED, "gmatrix: %zu rows are too many for a product's shared memory", w->rows);
    auto* q = new (std::nothrow) dz_cuda_gmatrix;
    if (!q) return fail(DZ_E_NOMEM, "host allocation");
    cudaStream_t st = nullptr;
    uint8_t *codes = nullptr, *scales = nullptr;
    int* bad = nullptr;
    const cudaError_t e = cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking);
    if (e != cudaSuccess) rc = gmv_fail("gmatrix: stream creation", e);
    if (!rc) rc = gmv_fill(w, &m, device, st, &codes, &scales, &bad);
    cudaFree(codes);
    cudaFree(scales);
    cudaFree(bad);
    if (st) cudaStreamDestroy(st);
    if (rc) {
        cudaFree(m.rec);
        delete q;
        return rc;
    }
    q->device = device;
    q->m = m;
    *out = q;
    return DZ_OK;
}

extern "C" void dz_cuda_gmatrix_free(dz_cuda_gmatrix_t* q) {
    if (!q) return;
    DeviceGuard g(q->device);
    cudaFree(q->m.rec);
    delete q;
}

extern "C" size_t dz_cuda_gmatrix_bytes(const dz_cuda_gmatrix_t* q) {
    return q ? (size_t)q->m.ntiles * q->m.nblocks * q->m.rec_bytes : 0;
}

extern "C" int dz_cuda_gmatrix_unpack(const dz_cuda_gmatrix_t* q, float* dst) {
    if (!q || !dst) return fail(DZ_E_INVALID, "null argument");
    DeviceGuard g(q->device);
    if (!g.ok) return fail(DZ_E_DEVICE, "cannot select device %d", q->device);
    const long long total = (long long)q->m.K * q->m.N;
    float* d = nullptr;
    DZ_CUDA(cudaMalloc(&d, total * 4));
    const unsigned grid = (unsigned)((total + 255) / 256);
    if (q->m.scale_f16)
        dz_gmv_dequant_kernel<__half><<<grid, 256>>>(q->m, d);
    else
        dz_gmv_dequant_kernel<float><<<grid, 256>>>(q->m, d);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaMemcpy(dst, d, total * 4, cudaMemcpyDeviceToHost);
    cudaFree(d);
    return e == cudaSuccess ? DZ_OK : gmv_fail("unpack", e);
}

extern "C" int dz_cuda_matmul_grouped_async(const void* A, size_t lda, const dz_cuda_gmatrix_t* q, void* C, size_t ldc,
                                            size_t m, size_t k, int type, void* stream) {
    if (!q || !A || !C) return fail(DZ_E_INVALID, "matmul_grouped: null argument");
    if (!type_ok(type)) return fail(DZ_E_INVALID, "matmul_grouped: unknown element type %d", type);
    if (m == 0 || m > (1u << 24) || k != (size_t)q->m.K)
        return fail(DZ_E_INVALID, "matmul_grouped: k must equal the matrix rows, m be 1..%u", 1u << 24);
    if (lda < k || ldc < (size_t)q->m.N || lda > (1ull << 40) || ldc > (1ull << 40))
        return fail(DZ_E_INVALID, "matmul_grouped: row strides must hold a row");
    if (((uintptr_t)A | (uintptr_t)C) % type_bytes(type))
        return fail(DZ_E_INVALID, "matmul_grouped: A and C must be aligned to their element type");
    DeviceGuard g(q->device);
    if (!g.ok) return fail(DZ_E_DEVICE, "cannot select device %d", q->device);
    GmvArgs a;
    a.w = q->m;
    a.x = A;
    a.y = C;
    a.ldx = (long long)lda;
    a.ldy = (long long)ldc;
    a.M = (int)m;
    a.type = type;
    DZ_CUDA(dz_gmv_launch(a, q->device, (cudaStream_t)stream));
    return DZ_OK;
}

extern "C" int dz_cuda_matmul_grouped(const float* A, const dz_cuda_gmatrix_t* q, float* C, size_t m, size_t k) {
    if (!q || !A || !C || m == 0 || m > (1u << 24) || k != (size_t)q->m.K)
        return fail(DZ_E_INVALID, "matmul_grouped: bad arguments (k must equal the matrix rows)");
    DeviceGuard g(q->device);
    if (!g.ok) return fail(DZ_E_DEVICE, "cannot select device %d", q->device);
    const size_t n = (size_t)q->m.N;
    float *dA = nullptr, *dC = nullptr;
    cudaError_t e = cudaMalloc(&dA, m * k * 4);
    if (e == cudaSuccess) e = cudaMalloc(&dC, m * n * 4);
    if (e == cudaSuccess) e = cudaMemcpy(dA, A, m * k * 4, cudaMemcpyHostToDevice);
    int rc = DZ_OK;
    if (e == cudaSuccess) rc = dz_cuda_matmul_grouped_async(dA, k, q, dC, n, m, k, DZ_TYPE_F32, nullptr);
    if (e == cudaSuccess && rc == DZ_OK) e = cudaMemcpy(C, dC, m * n * 4, cudaMemcpyDeviceToHost);
    cudaFree(dA);
    cudaFree(dC);
    if (rc) return rc;
    return e == cudaSuccess ? DZ_OK : gmv_fail("matmul_grouped", e);
}
