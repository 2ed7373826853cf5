// The 8-bit paged caches' append kernel (kv8.cuh) and C entry points.
#include "dz_cuda.h"

#include <atomic>
#include <cmath>

#include "headrows.cuh"
#include "kv4.cuh"
#include "kv8.cuh"
#include "shim.cuh"

namespace dz {

// A lane holds eight elements of a row in two quads that contain both elements
// of each pair of the rotation: element 8 l of 8 side by side, or 4 l of 4 of
// each half. Eight or sixteen lanes have a row, a warp four or two rows (or
// heads of one row).
//
// Many tokens: a block takes the new tokens of one sequence that fall in one
// page, and a share of their heads: keys, values, queries. A head's rows go to a
// team of 1 to 16 warps, four rows to a warp at most; a key or value head is
// held in registers until the team knows its peak, so that the page's scale
// needs no second pass over memory. The rows' angles are computed once per
// block: sine and cosine of every 8th row in 64 bits, the rows between by
// turning on by one token's angle (7 roundings of 2^-53).
//
// One token: a block takes a share of a row's heads, a warp two or four heads
// at a time.
//
// Queries are normed and rotated in fp32, as the scores that they enter are. Keys
// are in 64 bits up to one rounding to fp32, because the codes that follow round
// values next to a border and two summation orders would otherwise give different
// codes.

constexpr int KV8_WARPS = 16;      // warps of a block, many tokens
constexpr int KV8_ROWS = 4;        // rows of a warp
constexpr int KV8_ONE_WARPS = 8;   // warps of a block, one token
constexpr int KV8_QUERY_WARPS = 8; // warps of a block of queries
constexpr int KV8_TURN = 8;        // rows between angles that are computed afresh

struct Kv8AppendCut {
    int runs;                      // pages that a sequence's new tokens can touch
    int parts;                     // blocks that share a run's (a row's) heads
    int team;                      // warps of a head
};

template <typename T> union Kv8Quad {
    T e[4];
    uint2 w2;
    uint4 w4;
    __device__ Kv8Quad() {}
};

template <bool WIDE, typename T> __device__ __forceinline__ void kv8_load(const T* in, Kv8Quad<T>& to) {
    if (!WIDE) {
#pragma unroll
        for (int i = 0; i < 4; i++) to.e[i] = in[i];
    } else if (sizeof(T) == 4) {
        to.w4 = *reinterpret_cast<const uint4*>(in);
    } else {
        to.w2 = *reinterpret_cast<const uint2*>(in);
    }
}

template <bool WIDE, typename T> __device__ __forceinline__ void kv8_store(T* out, const float* x) {
    Kv8Quad<T> io;
#pragma unroll
    for (int i = 0; i < 4; i++) io.e[i] = dz_from_float<T>(x[i]);
    if (!WIDE) {
#pragma unroll
        for (int i = 0; i < 4; i++) out[i] = io.e[i];
    } else if (sizeof(T) == 4) {
        *reinterpret_cast<uint4*>(out) = io.w4;
    } else {
        *reinterpret_cast<uint2*>(out) = io.w2;
    }
}

// fp32 v rounded half away from zero and held to -127..127; a NaN gives 0.
__device__ __forceinline__ int kv8_round(float v) {
    const float r = __fadd_rn(v, copysignf(0.5f, v));
    return __float2int_rz(fminf(fmaxf(r, -127.0f), 127.0f)) & (v != v ? 0 : -1);
}
// The same for |v| <= 127 and two roundings.
__device__ __forceinline__ int kv8_round_held(float v) { return __float2int_rz(__fadd_rn(v, copysignf(0.5f, v))); }

// Turns the lane's four pairs by their angles.
template <typename A, typename C> __device__ __forceinline__ void kv8_rotate(A (&x)[8], bool halves, const C (&turn)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const A c = turn[i].x, s = turn[i].y;
        if (halves) {
            const A u = x[i], v = x[i + 4];
            x[i] = u * c - v * s;
            x[i + 4] = u * s + v * c;
        } else {
            const A u = x[2 * i], v = x[2 * i + 1];
            x[2 * i] = u * c - v * s;
            x[2 * i + 1] = u * s + v * c;
        }
    }
}

// A query's eight elements normed and rotated in fp32.
template <int HD>
__device__ __forceinline__ void kv8_query(float (&x)[8], const float (&gain)[8], const float2 (&turn)[4], const Kv8AppendArgs& a) {
    if (a.q_gain) {
        const float s = kv4_square_sum<HD / 8>(x, 0xffffffffu);
        float n = kv4_rsqrt(s * (1.0f / HD) + (float)a.eps);
        if (__any_sync(0xffffffffu, !(s > 1e-25f && s < 1e37f))) {   // squares that leave fp32's range
            double y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = (double)x[i];
            const double m = kv4_rsqrt(kv4_square_sum<HD / 8>(y, 0xffffffffu) / HD + a.eps);
            if (!(s > 1e-25f && s < 1e37f)) {
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = (float)(y[i] * m);
                n = 1.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = gain[i] * (x[i] * n);   // x n is about 1: gains of any size
    }
    if (a.rope) kv8_rotate(x, a.halves, turn);
}

// A key's eight elements, in 64 bits up to the last rounding; gain(i) is the gain
// of element i, turn(i) the angle of the i-th pair.
template <int HD, typename G, typename F>
__device__ __forceinline__ void kv8_key(float (&x)[8], G gain, F turn, const Kv8AppendArgs& a) {
    if (!a.k_gain && !a.rope) return;
    double y[8];
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = (double)x[i];
    if (a.k_gain) {
        const double n = kv4_rsqrt(kv4_square_sum<HD / 8>(y, 0xffffffffu) / HD + a.eps);
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = gain(i) * y[i] * n;
    }
    if (a.rope) {
        const double2 by[4] = {turn(0), turn(1), turn(2), turn(3)};
        kv8_rotate(y, a.halves, by);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)y[i];
}

__device__ __forceinline__ unsigned kv8_top(const float (&x)[8]) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    return top;
}

// The scale of a page's head from the new rows' largest magnitude (as bits;
// above 0x7f7fffff it is not finite) and the scale of the rows before them.
struct Kv8Scale {
    float scale, inverse;
    bool empty, plain;         // codes are 0; the codes need no clamp (not empty, and the inverse is finite)
};
__device__ __forceinline__ Kv8Scale kv8_scale(unsigned top, float old) {
    Kv8Scale s;
    const bool poisoned = top > 0x7f7fffffu || old != old;
    s.scale = poisoned ? __int_as_float(0x7fc00000) : fmaxf(old, __fdiv_rn(__uint_as_float(top), 127.0f));
    s.inverse = __fdiv_rn(1.0f, s.scale);
    s.empty = poisoned || s.scale == 0.0f;
    s.plain = s.scale >= 0x1p-120f;          // a peak's quotient rounds well there; false for a NaN
    return s;
}

// Codes of a lane's elements to the row at `to`; where `values` are wanted, x
// becomes what they stand for.
__device__ __forceinline__ void kv8_codes(float (&x)[8], const Kv8Scale& s, int8_t* to, const int (&at)[2], bool values) {
#pragma unroll
    for (int q = 0; q < 2; q++) {
        int c[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float v = __fmul_rn(x[4 * q + i], s.inverse);
            c[i] = s.plain ? kv8_round_held(v) : s.empty ? 0 : kv8_round(v);
        }
        *reinterpret_cast<unsigned*>(to + at[q]) = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
        if (values) {
            // 2^23 + 2^22 + c, less 2^23 + 2^22
#pragma unroll
            for (int i = 0; i < 4; i++) x[4 * q + i] = (__int_as_float(0x4B400000 + c[i]) - 12582912.0f) * s.scale;
        }
    }
}

// The codes of a page's first `rows` rows after its scale went from `old` to
// `scale`: thread `me` of `count`.
template <int HD> __device__ __forceinline__ void kv8_rescale(int8_t* codes, int rows, float old, float scale, int me, int count) {
    const float ratio = __fdiv_rn(old, scale);
    for (int i = me; i < rows * (HD / 16); i += count) {
        uint4* at = reinterpret_cast<uint4*>(codes) + i;
        uint4 v = *at;
        unsigned* w = reinterpret_cast<unsigned*>(&v);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            unsigned n = 0;
#pragma unroll
            for (int e = 0; e < 4; e++)
                n |= ((unsigned)kv8_round(__fmul_rn((float)(int)(int8_t)(w[q] >> (8 * e)), ratio)) & 0xffu) << (8 * e);
            w[q] = n;
        }
        *at = v;
    }
}

// Where the angle of pair p of a row lies: the i-th pairs of a row's lanes side by side.
template <int HD> __device__ __forceinline__ int kv8_angle_at(int p) { return p % 4 * (HD / 8) + p / 4; }

template <typename T, int HD, bool WIDE>     // every row of every operand is aligned to a quad
__global__ void __launch_bounds__(KV8_WARPS * 32, 2) dz_kv8_append_kernel(const __grid_constant__ Kv8AppendArgs a,
                                                                         const __grid_constant__ Kv8AppendCut cut) {
    constexpr int LANES = HD / 8, SLOTS = 32 / LANES, R = KV8_ROWS / SLOTS, P = HD / 2;
    extern __shared__ __align__(16) double2 kv8_angles[];                          // [rows][P]
    __shared__ unsigned tops[2][KV8_WARPS];
    __shared__ __align__(16) double gains[HD];
    asm volatile("griddepcontrol.wait;" ::: "memory");   // launched while the kernel before ends
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % LANES, slot = lane / LANES;
    const int at[2] = {a.halves ? l * 4 : l * 8, a.halves ? P + l * 4 : l * 8 + 4};
    int where = blockIdx.x;
    const int part = where % cut.parts;
    where /= cut.parts;
    const int run = where % cut.runs, b = where / cut.runs;
    const long long first = a.positions[b];
    if (kv8_skips(first)) return;
    // this block's tokens: lo..hi-1 of the call's, all in page `j` of the sequence
    const long long j = first / a.c.page + run, start = j * a.c.page;
    const int lo = (int)max(0LL, start - first), hi = (int)min((long long)a.n_tokens, start + a.c.page - first);
    if (lo >= hi) return;
    const int rows = hi - lo, offset = (int)(first + lo - start);     // rows of the page before them
    int page = -1;
    if (j < a.c.table_pages) page = a.c.table[(long long)b * a.c.table_pages + j];
    const bool held = (unsigned)page < (unsigned)a.c.pages;
    if (a.rope) {
        for (int i = threadIdx.x; i < P * ((rows + KV8_TURN - 1) / KV8_TURN); i += KV8_WARPS * 32) {
            const int p = i % P, r0 = i / P * KV8_TURN, r1 = min(r0 + KV8_TURN, rows);
            double c, s, c1, s1;
            sincos((double)(first + lo + r0) * a.freq[p], &s, &c);
            sincos(a.freq[p], &s1, &c1);
            for (int r = r0; r < r1; r++) {
                kv8_angles[r * P + kv8_angle_at<HD>(p)] = make_double2(c, s);
                const double next = c * c1 - s * s1;
                s = s * c1 + c * s1;
                c = next;
            }
        }
    }
    if (a.k_gain)
        for (int i = threadIdx.x; i < HD; i += KV8_WARPS * 32) gains[i] = (double)a.k_gain[i];
    __syncthreads();
    const int team = cut.team, mine = warp / team, rank = warp % team, teams = KV8_WARPS / team;
    const int step = cut.parts * teams, heads = 2 * a.c.kv_heads;
    const long long row0 = (long long)b * a.n_tokens + lo;
    // the warp's rows: SLOTS at a time, those of the team in turn
    auto row_of = [&](int i) { return (i * team + rank) * SLOTS + slot; };
    auto load = [&](int item, Kv8Quad<T> (&io)[R][2]) {
        if (item >= heads) return;
        const bool key = item < a.c.kv_heads;
        const long long ld = key ? a.ldk : a.ldv;
        const T* in = static_cast<const T*>(key ? a.k : a.v) + row0 * ld + (key ? item : item - a.c.kv_heads) * HD;
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int r = row_of(i);
            if (r < rows) {
                kv8_load<WIDE>(in + r * ld + at[0], io[i][0]);
                kv8_load<WIDE>(in + r * ld + at[1], io[i][1]);
            }
        }
    };
    int item = part * teams + mine, parity = 0;
    Kv8Quad<T> next[R][2];
    load(item, next);
    float x[R][8];
    auto take = [&] {                        // the item's elements, and the next one's loads
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[i][e] = row_of(i) < rows ? dz_to_float(next[i][e / 4].e[e % 4]) : 0.0f;
        load(item + step, next);
    };
    for (; item < heads; item += step) {
        take();
        if (!held) continue;                 // the whole block alike
        const bool key = item < a.c.kv_heads;
        const int h = key ? item : item - a.c.kv_heads;
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int r = min(row_of(i), rows - 1);
            if (key && (i * team + rank) * SLOTS < rows)                 // the warp alike
                kv8_key<HD>(x[i], [&](int e) { return gains[at[e / 4] + e % 4]; },
                            [&](int p) { return kv8_angles[r * P + p * LANES + l]; }, a);
            if (row_of(i) < rows) top = max(top, kv8_top(x[i]));
        }
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
        const long long place = (long long)page * a.c.kv_heads + h;      // the page's head
        float* scales = key ? a.c.k_scales : a.c.v_scales;
        const float old = offset ? scales[place] : 0.0f;
        if (team > 1) {                      // the team's peak
            if (lane == 0) tops[parity][warp] = top;
            asm volatile("bar.sync %0, %1;" ::"r"(mine + 1), "r"(team * 32) : "memory");
            for (int w = 0; w < team; w++) top = max(top, tops[parity][mine * team + w]);
            parity ^= 1;                     // read by all before the team's next barrier but one
        } else {
            __syncwarp();
        }
        const Kv8Scale s = kv8_scale(top, old);
        int8_t* codes = (key ? a.c.k_codes : a.c.v_codes) + place * (a.c.page * HD);
        if (offset && s.scale > old) kv8_rescale<HD>(codes, offset, old, s.scale, rank * 32 + lane, team * 32);
        if (rank == 0 && lane == 0) scales[place] = s.scale;
        T* out = static_cast<T*>(key ? a.k_out : a.v_out);
        const long long ldo = key ? a.ldko : a.ldvo;
        if (out) out += row0 * ldo + h * HD;
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int r = row_of(i);
            if (r >= rows) continue;
            kv8_codes(x[i], s, codes + (offset + r) * HD, at, out != nullptr);
            if (out) {
                kv8_store<WIDE>(out + r * ldo + at[0], x[i]);
                kv8_store<WIDE>(out + r * ldo + at[1], x[i] + 4);
            }
        }
    }
}

// Queries of many tokens: a warp takes SLOTS rows, whose angles and gains stay in
// registers, and a share of their heads in turn. Where rows are aligned, the heads
// after it are on their way into shared memory, each lane copying what it reads
// itself.
template <typename T> struct Kv8Ring {
    static constexpr int HEADS = 8;                    // of a warp's rows, in turn
    static constexpr int SMEM = HEADS * KV8_QUERY_WARPS * 32 * (int)(2 * sizeof(Kv8Quad<T>));
};

template <typename T, int HD, bool WIDE>
__global__ void __launch_bounds__(KV8_QUERY_WARPS * 32, 3) dz_kv8_query_kernel(const __grid_constant__ Kv8AppendArgs a, int parts) {
    constexpr int LANES = HD / 8, SLOTS = 32 / LANES, P = HD / 2, HEADS = Kv8Ring<T>::HEADS, B = 4 * (int)sizeof(T);
    extern __shared__ __align__(16) uint8_t kv8_heads[];           // [HEADS][2 quads][threads]
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, l = lane % LANES, slot = lane / LANES;
    const int work = blockIdx.x * KV8_QUERY_WARPS + (threadIdx.x >> 5), set = work / parts, part = work % parts;
    const int rows = a.c.batch * a.n_tokens;
    if (set * SLOTS >= rows) return;
    const int row = min(set * SLOTS + slot, rows - 1), b = row / a.n_tokens;
    const long long first = a.positions[b];
    const bool done = set * SLOTS + slot < rows && !kv8_skips(first);
    const int at = a.halves ? l * 4 : l * 8, quad = a.halves ? P : 4;
    const int h0 = a.q_heads * part / parts, n = a.q_heads * (part + 1) / parts - h0;
    const T* in = static_cast<const T*>(a.q) + row * a.ldq + h0 * HD + at;
    T* out = static_cast<T*>(a.q_out) + row * a.ldqo + h0 * HD + at;
    auto place = [&](int k, int q) { return kv8_heads + ((k * 2 + q) * (KV8_QUERY_WARPS * 32) + (int)threadIdx.x) * B; };
    auto copy = [&](int k, int h) {
        if (h < n) {
#pragma unroll
            for (int q = 0; q < 2; q++)
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(place(k, q))),
                             "l"(in + h * HD + q * quad), "n"(B)
                             : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (WIDE) {
#pragma unroll
        for (int k = 0; k < HEADS - 1; k++) copy(k, k);
    }
    float2 turn[4];
#pragma unroll
    for (int p = 0; p < 4; p++)
        if (a.rope) {
            double c, s;
            sincos((double)(first + (row - b * a.n_tokens)) * a.freq[l * 4 + p], &s, &c);
            turn[p] = make_float2((float)c, (float)s);
        }
    float gain[8];
#pragma unroll
    for (int i = 0; i < 8; i++) gain[i] = a.q_gain ? a.q_gain[at + i / 4 * quad + i % 4] : 1.0f;
#pragma unroll 1
    for (int h = 0; h < n; h++) {
        Kv8Quad<T> io[2];
        if (WIDE) {
            copy((h + HEADS - 1) % HEADS, h + HEADS - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(HEADS - 1) : "memory");
#pragma unroll
            for (int q = 0; q < 2; q++) kv8_load<true>(reinterpret_cast<const T*>(place(h % HEADS, q)), io[q]);
        } else {
            kv8_load<false>(in + h * HD, io[0]);
            kv8_load<false>(in + h * HD + quad, io[1]);
        }
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = dz_to_float(io[e / 4].e[e % 4]);
        kv8_query<HD>(y, gain, turn, a);
        if (done) {
            kv8_store<WIDE>(out + h * HD, y);
            kv8_store<WIDE>(out + h * HD + quad, y + 4);
        }
    }
}

// One new token of every sequence.
template <typename T, int HD, bool WIDE>
__global__ void __launch_bounds__(KV8_ONE_WARPS * 32, 4) dz_kv8_append_one_kernel(const __grid_constant__ Kv8AppendArgs a,
                                                                             const __grid_constant__ Kv8AppendCut cut) {
    constexpr int LANES = HD / 8, SLOTS = 32 / LANES, P = HD / 2;
    __shared__ double2 angles[P];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % LANES, slot = lane / LANES;
    const int at[2] = {a.halves ? l * 4 : l * 8, a.halves ? P + l * 4 : l * 8 + 4};
    const int b = blockIdx.x / (unsigned)cut.parts, part = blockIdx.x % (unsigned)cut.parts;
    const long long pos = a.positions[b];
    const int nk = (a.c.kv_heads + SLOTS - 1) / SLOTS, nq = (a.q_heads + SLOTS - 1) / SLOTS;    // items
    const int step = cut.parts * KV8_ONE_WARPS;
    Kv8Quad<T> next[2];
    auto load = [&](int item) {              // keys, then values, then queries
        const bool key = item < nk, value = !key && item < 2 * nk;
        const int h = (key ? item : value ? item - nk : item - 2 * nk) * SLOTS + slot;
        if (item >= 2 * nk + nq || h >= (key || value ? a.c.kv_heads : a.q_heads)) return;
        const T* in = static_cast<const T*>(key ? a.k : value ? a.v : a.q) + b * (key ? a.ldk : value ? a.ldv : a.ldq) + h * HD;
        kv8_load<WIDE>(in + at[0], next[0]);
        kv8_load<WIDE>(in + at[1], next[1]);
    };
    int item = part * KV8_ONE_WARPS + warp;
    load(item);
    if (kv8_skips(pos)) return;
    const long long j = pos / a.c.page;
    const int offset = (int)(pos - j * a.c.page);        // rows of the page before the token's
    int page = -1;
    if (j < a.c.table_pages) page = a.c.table[(long long)b * a.c.table_pages + j];
    const bool held = (unsigned)page < (unsigned)a.c.pages;
    if (a.rope) {
        if (threadIdx.x < P) {
            double c, s;
            sincos((double)pos * a.freq[threadIdx.x], &s, &c);
            angles[kv8_angle_at<HD>(threadIdx.x)] = make_double2(c, s);
        }
        __syncthreads();
    }
    float x[8], gain[8];
    auto gains = [&](const float* g) {
#pragma unroll
        for (int i = 0; i < 8; i++) gain[i] = g ? g[at[i / 4] + i % 4] : 1.0f;
    };
    if (item < nk) gains(a.k_gain);
    auto take = [&](bool valid) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = valid ? dz_to_float(next[e / 4].e[e % 4]) : 0.0f;
        load(item + step);
    };
    for (; item < 2 * nk; item += step) {
        const bool key = item < nk;
        const int h = (key ? item : item - nk) * SLOTS + slot;
        const bool valid = h < a.c.kv_heads;
        take(valid);
        if (!held) continue;
        const long long place = (long long)page * a.c.kv_heads + (valid ? h : 0);
        float* scales = key ? a.c.k_scales : a.c.v_scales;
        const float old = offset ? scales[place] : 0.0f;
        if (key) kv8_key<HD>(x, [&](int e) { return (double)gain[e]; }, [&](int p) { return angles[p * LANES + l]; }, a);
        unsigned top = kv8_top(x);
#pragma unroll
        for (int off = LANES / 2; off >= 1; off >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
        __syncwarp();                        // every lane has the old scale
        if (!valid) continue;
        const Kv8Scale s = kv8_scale(top, old);
        int8_t* codes = (key ? a.c.k_codes : a.c.v_codes) + place * (a.c.page * HD);
        if (offset && s.scale > old) kv8_rescale<HD>(codes, offset, old, s.scale, l, LANES);
        if (l == 0) scales[place] = s.scale;
        T* out = static_cast<T*>(key ? a.k_out : a.v_out);
        kv8_codes(x, s, codes + offset * HD, at, out != nullptr);
        if (out) {
            out += b * (key ? a.ldko : a.ldvo) + h * HD;
            kv8_store<WIDE>(out + at[0], x);
            kv8_store<WIDE>(out + at[1], x + 4);
        }
    }
    if (item < 2 * nk + nq) gains(a.q_gain);
    for (; item < 2 * nk + nq; item += step) {
        const int h = (item - 2 * nk) * SLOTS + slot;
        take(h < a.q_heads);
        float2 turn[4];
#pragma unroll
        for (int p = 0; p < 4; p++)
            if (a.rope) {
                const double2 d = angles[p * LANES + l];
                turn[p] = make_float2((float)d.x, (float)d.y);
            }
        kv8_query<HD>(x, gain, turn, a);
        if (h < a.q_heads) {
            T* out = static_cast<T*>(a.q_out) + b * a.ldqo + h * HD;
            kv8_store<WIDE>(out + at[0], x);
            kv8_store<WIDE>(out + at[1], x + 4);
        }
    }
}

constexpr int KV8_DEVICES = 64;

template <typename T, int HD, bool WIDE> static cudaError_t kv8_append_t(const Kv8AppendArgs& a, int device, int sms, cudaStream_t st) {
    static std::atomic<bool> ready[KV8_DEVICES];
    const int rows = a.n_tokens < a.c.page ? a.n_tokens : a.c.page;          // of a block at most
    Kv8AppendCut cut;
    long long blocks = a.c.batch, most;                  // most: blocks that have heads for their warps
    if (a.n_tokens == 1) {
        constexpr int SLOTS = 256 / HD;
        cut.runs = cut.team = 1;
        most = (2 * ((a.c.kv_heads + SLOTS - 1) / SLOTS) + (a.q_heads + SLOTS - 1) / SLOTS + KV8_ONE_WARPS - 1) / KV8_ONE_WARPS;
    } else {
        cut.runs = (int)(((long long)a.n_tokens + a.c.page - 2) / a.c.page) + 1;
        blocks *= cut.runs;
        for (cut.team = 1; cut.team * KV8_ROWS < rows;) cut.team *= 2;
        const int teams = KV8_WARPS / cut.team;
        most = (2 * a.c.kv_heads + teams - 1) / teams;
    }
    // as many blocks as the SMs hold at once (four, two of many tokens), as far as there are heads: a part of a wave
    // more cost 8000 rows a third of their time
    const long long parts = (a.n_tokens == 1 ? 4LL : 2LL) * sms / blocks;
    cut.parts = (int)(parts < 1 ? 1 : parts < most ? parts : most);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(blocks * cut.parts));
    cfg.blockDim = dim3((a.n_tokens == 1 ? KV8_ONE_WARPS : KV8_WARPS) * 32);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (a.n_tokens == 1) return cudaLaunchKernelEx(&cfg, dz_kv8_append_one_kernel<T, HD, WIDE>, a, cut);
    constexpr int most_smem = 64 * (HD / 2) * (int)sizeof(double2);
    if (!ready[device].load(std::memory_order_acquire)) {
        const cudaError_t set = cudaFuncSetAttribute(dz_kv8_append_kernel<T, HD, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, most_smem);
        if (set != cudaSuccess) return set;
        const cudaError_t ring = cudaFuncSetAttribute(dz_kv8_query_kernel<T, HD, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Kv8Ring<T>::SMEM);
        if (ring != cudaSuccess) return ring;
        ready[device].store(true, std::memory_order_release);
    }
    cfg.dynamicSmemBytes = a.rope ? (size_t)rows * (HD / 2) * sizeof(double2) : 0;
    cudaError_t e = cudaLaunchKernelEx(&cfg, dz_kv8_append_kernel<T, HD, WIDE>, a, cut);
    if (e != cudaSuccess || a.q_heads == 0) return e;
    // sets of rows that a warp takes, and its share of their heads where there are few
    const long long sets = ((long long)a.c.batch * a.n_tokens + 256 / HD - 1) / (256 / HD), fit = 3LL * sms * KV8_QUERY_WARPS;
    const long long share = (fit + sets - 1) / sets;
    const int query_parts = (int)(share < a.q_heads ? share : a.q_heads);
    cfg.gridDim = dim3((unsigned)((sets * query_parts + KV8_QUERY_WARPS - 1) / KV8_QUERY_WARPS));
    cfg.blockDim = dim3(KV8_QUERY_WARPS * 32);
    cfg.dynamicSmemBytes = WIDE ? Kv8Ring<T>::SMEM : 0;
    return cudaLaunchKernelEx(&cfg, dz_kv8_query_kernel<T, HD, WIDE>, a, query_parts);
}

template <typename T> static cudaError_t kv8_append_h(const Kv8AppendArgs& a, int head_dim, int device, int sms, cudaStream_t st) {
    const uintptr_t bases = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.k_out |
                            (uintptr_t)a.v_out;
    const long long strides = a.ldq | a.ldk | a.ldv | a.ldqo | a.ldko | a.ldvo;
    if (bases % (4 * sizeof(T)) == 0 && strides % 4 == 0)
        return head_dim == 128 ? kv8_append_t<T, 128, true>(a, device, sms, st) : kv8_append_t<T, 64, true>(a, device, sms, st);
    return head_dim == 128 ? kv8_append_t<T, 128, false>(a, device, sms, st) : kv8_append_t<T, 64, false>(a, device, sms, st);
}

cudaError_t dz_kv8_append_launch(const Kv8AppendArgs& a, int type, int head_dim, int device, cudaStream_t st) {
    if (device < 0 || device >= KV8_DEVICES) return cudaErrorInvalidDevice;
    static std::atomic<int> known[KV8_DEVICES];       // SM count per device, looked up once
    int sms = known[device].load(std::memory_order_relaxed);
    if (!sms) {
        const cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
        if (e != cudaSuccess) return e;
        known[device].store(sms, std::memory_order_relaxed);
    }
    if (type == DZ_TYPE_F32) return kv8_append_h<float>(a, head_dim, device, sms, st);
    if (type == DZ_TYPE_F16) return kv8_append_h<__half>(a, head_dim, device, sms, st);
    return kv8_append_h<__nv_bfloat16>(a, head_dim, device, sms, st);
}

}  // namespace dz

using namespace dz;

// The limits keep every index of a launch in range: rows x heads below 2^31, a
// code buffer (pages x heads x 64 x 128 bytes) below 2^60.
static int kv8_check(const dz_kv8_t* c, const int64_t* positions, size_t n_tokens, Kv8Cache* out) {
    if (!c || !c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales || !c->table || !positions)
        return fail(DZ_E_INVALID, "kv8: null argument");
    if (c->head_dim != 64 && c->head_dim != 128)
        return fail(DZ_E_UNSUPPORTED, "kv8: head dimension %zu (64 and 128 are supported)", c->head_dim);
    if (c->page != 32 && c->page != 64)
        return fail(DZ_E_UNSUPPORTED, "kv8: pages of %zu tokens (32 and 64 are supported)", c->page);
    if (c->batch == 0 || c->batch > 65535 || c->kv_heads == 0 || c->kv_heads > 65535)
        return fail(DZ_E_INVALID, "kv8: batch and kv_heads must be 1..65535");
    if (c->pages == 0 || c->pages > (size_t)INT32_MAX) return fail(DZ_E_INVALID, "kv8: pages must be 1..2^31-1");
    if (c->table_pages == 0 || c->table_pages > (size_t)KV8_REACH / c->page)
        return fail(DZ_E_INVALID, "kv8: table_pages must be 1 and more, and its positions at most 2^31 - 64");
    if (n_tokens == 0 || n_tokens > c->table_pages * c->page)
        return fail(DZ_E_INVALID, "kv8: n_tokens must be 1..table_pages * page (%zu)", c->table_pages * c->page);
    if ((((uintptr_t)c->k_codes | (uintptr_t)c->v_codes) & 15) ||
        (((uintptr_t)c->k_scales | (uintptr_t)c->v_scales | (uintptr_t)c->table) & 3) || ((uintptr_t)positions & 7))
        return fail(DZ_E_INVALID, "kv8: code buffers must be 16-byte aligned, scales and the table 4-byte, positions 8-byte");
    *out = Kv8Cache{c->k_codes,       c->v_codes,        c->k_scales,   c->v_scales,  c->table,
                    (int)c->batch,    (int)c->kv_heads,  (int)c->pages, (int)c->page, (int)c->table_pages};
    return DZ_OK;
}

// A typed row-strided operand: base aligned to its type, rows that hold their
// heads, offsets in range.
static int kv8_rows(const char* what, const void* base, size_t stride, size_t heads, size_t head_dim, int type) {
    if (!base) return fail(DZ_E_INVALID, "kv8: %s is null", what);
    if ((uintptr_t)base % type_bytes(type)) return fail(DZ_E_INVALID, "kv8: %s is not aligned to its type", what);
    if (stride < heads * head_dim || stride > (1ull << 40))
        return fail(DZ_E_INVALID, "kv8: %s rows of %zu elements do not hold %zu heads", what, stride, heads);
    return DZ_OK;
}

extern "C" int dz_cuda_kv8_append(const dz_kv8_t* c, const dz_kv8_append_t* p, const int64_t* positions, size_t n_tokens,
                                  void* stream) {
    Kv8AppendArgs a;
    if (!p) return fail(DZ_E_INVALID, "kv8: null argument");
    int rc = kv8_check(c, positions, n_tokens, &a.c);
    if (rc) return rc;
    if (!type_ok(p->type)) return fail(DZ_E_INVALID, "kv8: unknown element type %d", p->type);
    // as many blocks as pages of new tokens (one more than they fill) and heads, all below 2^31
    if (p->q_heads > 65535 ||
        c->batch * (n_tokens + c->page) > (size_t)INT32_MAX / (p->q_heads + 2 * c->kv_heads))
        return fail(DZ_E_INVALID, "kv8: too many rows x heads in one call");
    if (p->q_heads) {
        if ((rc = kv8_rows("q", p->q, p->q_stride, p->q_heads, c->head_dim, p->type))) return rc;
        if ((rc = kv8_rows("q_out", p->q_out, p->q_out_stride, p->q_heads, c->head_dim, p->type))) return rc;
    }
    if ((rc = kv8_rows("k", p->k, p->k_stride, c->kv_heads, c->head_dim, p->type))) return rc;
    if ((rc = kv8_rows("v", p->v, p->v_stride, c->kv_heads, c->head_dim, p->type))) return rc;
    if (p->k_out && (rc = kv8_rows("k_out", p->k_out, p->k_out_stride, c->kv_heads, c->head_dim, p->type))) return rc;
    if (p->v_out && (rc = kv8_rows("v_out", p->v_out, p->v_out_stride, c->kv_heads, c->head_dim, p->type))) return rc;
    if ((p->q_gain || p->k_gain) && !(p->eps >= 0.0 && std::isfinite(p->eps)))
        return fail(DZ_E_INVALID, "kv8: the norm's eps must be finite and >= 0");
    if (((uintptr_t)p->q_gain | (uintptr_t)p->k_gain) & 3) return fail(DZ_E_INVALID, "kv8: gains are not aligned");
    if (p->rope_base != 0.0 && !(p->rope_base > 0.0 && std::isfinite(p->rope_base)))
        return fail(DZ_E_INVALID, "kv8: rope_base must be 0 (no rotation) or positive");
    if (p->rope_pairing != DZ_ROPE_PAIRS && p->rope_pairing != DZ_ROPE_HALVES)
        return fail(DZ_E_INVALID, "kv8: unknown rotation pairing %d", p->rope_pairing);
    DeviceGuard g(c->device);
    if (!g.ok) return fail(DZ_E_DEVICE, "cannot select device %d", c->device);
    a.positions = (const long long*)positions;
    a.q = p->q_heads ? p->q : nullptr;
    a.k = p->k;
    a.v = p->v;
    a.q_out = p->q_heads ? p->q_out : nullptr;
    a.k_out = p->k_out;
    a.v_out = p->v_out;
    a.ldq = p->q_heads ? (long long)p->q_stride : 0;
    a.ldk = (long long)p->k_stride;
    a.ldv = (long long)p->v_stride;
    a.ldqo = p->q_heads ? (long long)p->q_out_stride : 0;
    a.ldko = p->k_out ? (long long)p->k_out_stride : 0;
    a.ldvo = p->v_out ? (long long)p->v_out_stride : 0;
    a.q_gain = p->q_gain;
    a.k_gain = p->k_gain;
    a.eps = p->eps;
    a.n_tokens = (int)n_tokens;
    a.q_heads = (int)p->q_heads;
    a.rope = p->rope_base != 0.0;
    a.halves = p->rope_pairing == DZ_ROPE_HALVES;
    dz_kv4_frequencies(p->rope_base, c->head_dim, a.freq);
    DZ_CUDA(dz_kv8_append_launch(a, p->type, (int)c->head_dim, c->device, (cudaStream_t)stream));
    return DZ_OK;
}

extern "C" int dz_cuda_kv8_attention(const dz_kv8_t* c, const dz_kv8_attention_t* p, const int64_t* positions,
                                     size_t n_tokens, void* stream) {
    Kv8AttnArgs a;
    if (!p) return fail(DZ_E_INVALID, "kv8: null argument");
    int rc = kv8_check(c, positions, n_tokens, &a.c);
    if (rc) return rc;
    if (!type_ok(p->type)) return fail(DZ_E_INVALID, "kv8: unknown element type %d", p->type);
    if (p->q_heads == 0 || p->q_heads > 65535 || p->q_heads % c->kv_heads)
        return fail(DZ_E_INVALID, "kv8: q_heads must be a multiple of kv_heads");
    if (c->batch * n_tokens > (size_t)INT32_MAX / 16 / p->q_heads)
        return fail(DZ_E_INVALID, "kv8: too many rows x heads in one call");
    if ((rc = kv8_rows("q", p->q, p->q_stride, p->q_heads, c->head_dim, p->type))) return rc;
    if ((rc = kv8_rows("out", p->out, p->out_stride, p->q_heads, c->head_dim, p->type))) return rc;
    if (!std::isfinite(p->scale)) return fail(DZ_E_INVALID, "kv8: scale must be finite");
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
    const long long reach = (long long)a.c.table_pages * a.c.page;
    a.window = p->window < ((size_t)1 << 62) ? (long long)p->window : 1LL << 62;
    const long long longest = p->longest && p->longest < (size_t)reach ? (long long)p->longest : reach;
    DZ_CUDA(dz_kv8_attn_launch(a, longest, p->type, (int)c->head_dim, c->device, (cudaStream_t)stream));
    return DZ_OK;
}
