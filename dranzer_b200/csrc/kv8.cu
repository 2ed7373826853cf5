// The 8-bit paged caches' append kernel (kv8.cuh) and C entry points.
#include "dz_cuda.h"

#include <atomic>
#include <cmath>

#include "headrows.cuh"
#include "kv4.cuh"
#include "kv8.cuh"
#include "shim.cuh"

namespace dz {

// A block takes the new tokens of one sequence that fall in one page, and a
// share of their heads: keys, values, queries. A head's rows go to a team of 1
// to 8 warps, at most eight rows to a warp, a row over the lanes of a warp; a
// key or value head is held in registers until the team knows its peak, so that
// the page's scale needs no second pass over memory. The rows' angles are
// computed once per block: sine and cosine of every 16th row in 64 bits, the
// rows between by turning on by one token's angle (15 roundings of 2^-53).
//
// Queries are normed and rotated in fp32. Keys are in 64 bits up to one
// rounding to fp32, because the codes that follow round values next to a border
// and two summation orders would otherwise give different codes.

constexpr int KV8_WARPS = 8;
constexpr int KV8_ROWS = 8;        // rows of a warp
constexpr int KV8_TURN = 16;       // rows between angles that are computed afresh

struct Kv8AppendCut {
    int runs;                      // pages that a sequence's new tokens can touch
    int parts;                     // blocks that share a run's heads
    int team;                      // warps of a head
    int wide;                      // every row of every operand is aligned to a lane's elements
    int table_rows;                // rows of the angle table
};

template <typename T, int E> union Kv8Lane {     // a lane's elements of a row
    T e[E];
    uint2 w2;
    uint4 w4;
    unsigned w1;
    __device__ Kv8Lane() {}
};

template <typename T, int E> __device__ __forceinline__ void kv8_load(const T* in, bool wide, Kv8Lane<T, E>& to) {
    constexpr int B = E * (int)sizeof(T);
    if (!wide) {
#pragma unroll
        for (int i = 0; i < E; i++) to.e[i] = in[i];
    } else if (B == 16) {
        to.w4 = *reinterpret_cast<const uint4*>(in);
    } else if (B == 8) {
        to.w2 = *reinterpret_cast<const uint2*>(in);
    } else {
        to.w1 = *reinterpret_cast<const unsigned*>(in);
    }
}

template <typename T, int E> __device__ __forceinline__ void kv8_store(T* out, bool wide, const float (&x)[E]) {
    constexpr int B = E * (int)sizeof(T);
    Kv8Lane<T, E> io;
#pragma unroll
    for (int i = 0; i < E; i++) io.e[i] = dz_from_float<T>(x[i]);
    if (!wide) {
#pragma unroll
        for (int i = 0; i < E; i++) out[i] = io.e[i];
    } else if (B == 16) {
        *reinterpret_cast<uint4*>(out) = io.w4;
    } else if (B == 8) {
        *reinterpret_cast<uint2*>(out) = io.w2;
    } else {
        *reinterpret_cast<unsigned*>(out) = io.w1;
    }
}

// fp32 v rounded half away from zero and held to -127..127; a NaN gives 0.
__device__ __forceinline__ int kv8_round(float v) {
    const float r = __fadd_rn(v, copysignf(0.5f, v));
    return __float2int_rz(fminf(fmaxf(r, -127.0f), 127.0f)) & (v != v ? 0 : -1);
}

template <typename T, int HD>
__global__ void __launch_bounds__(KV8_WARPS * 32) dz_kv8_append_kernel(const __grid_constant__ Kv8AppendArgs a,
                                                                      const __grid_constant__ Kv8AppendCut cut) {
    constexpr int E = HD / 32, P = HD / 2;
    extern __shared__ __align__(16) uint8_t kv8_smem[];
    double2* angles = reinterpret_cast<double2*>(kv8_smem);                        // [rows][P]
    float2* angles_f = reinterpret_cast<float2*>(angles + cut.table_rows * P);     // [rows][P]
    __shared__ unsigned tops[2][KV8_WARPS];
    asm volatile("griddepcontrol.wait;" ::: "memory");   // launched while the kernel before ends
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, at = lane * E;
    int where = blockIdx.x;
    const int part = where % cut.parts;
    where /= cut.parts;
    const int run = where % cut.runs, b = where / cut.runs;
    const long long first = a.positions[b];
    if (kv8_skips(first)) return;
    // this block's tokens: lo..hi-1 of the call's, all in page `slot` of the sequence
    const long long slot = first / a.c.page + run, start = slot * a.c.page;
    const int lo = (int)max(0LL, start - first), hi = (int)min((long long)a.n_tokens, start + a.c.page - first);
    if (lo >= hi) return;
    const int rows = hi - lo, offset = (int)(first + lo - start);     // rows of the page before them
    int where_page = -1;
    if (slot < a.c.table_pages) where_page = a.c.table[(long long)b * a.c.table_pages + slot];
    const bool held = (unsigned)where_page < (unsigned)a.c.pages;
    if (a.rope) {
        for (int i = threadIdx.x; i < P * ((rows + KV8_TURN - 1) / KV8_TURN); i += KV8_WARPS * 32) {
            const int p = i % P, r0 = i / P * KV8_TURN, r1 = min(r0 + KV8_TURN, rows);
            double c, s, c1, s1;
            sincos((double)(first + lo + r0) * a.freq[p], &s, &c);
            sincos(a.freq[p], &s1, &c1);
            for (int r = r0; r < r1; r++) {
                angles[r * P + p] = make_double2(c, s);
                angles_f[r * P + p] = make_float2((float)c, (float)s);
                const double next = c * c1 - s * s1;
                s = s * c1 + c * s1;
                c = next;
            }
        }
        __syncthreads();
    }
    const int team = cut.team, mine = warp / team, rank = warp % team, teams = KV8_WARPS / team;
    const int step = cut.parts * teams;
    const long long row0 = (long long)b * a.n_tokens + lo;
    // the lane's pair i of a row: (2p, 2p + 1), or element e with e + HD / 2
    const int pair0 = a.halves ? at % P : at / 2;
    int parity = 0;
    for (int item = part * teams + mine; item < 2 * a.c.kv_heads + a.q_heads; item += step) {
        if (item >= 2 * a.c.kv_heads) {      // a query head
            const int h = item - 2 * a.c.kv_heads;
            const T* in = static_cast<const T*>(a.q) + row0 * a.ldq + h * HD + at;
            T* out = static_cast<T*>(a.q_out) + row0 * a.ldqo + h * HD + at;
            float gain[E];
#pragma unroll
            for (int i = 0; i < E; i++) gain[i] = a.q_gain ? a.q_gain[at + i] : 1.0f;
            Kv8Lane<T, E> io[KV8_ROWS];
#pragma unroll
            for (int j = 0; j < KV8_ROWS; j++) {
                const int r = rank + j * team;
                if (r < rows) kv8_load<T, E>(in + r * a.ldq, cut.wide, io[j]);
            }
#pragma unroll
            for (int j = 0; j < KV8_ROWS; j++) {
                const int r = rank + j * team;
                if (r >= rows) break;
                float x[E];
#pragma unroll
                for (int i = 0; i < E; i++) x[i] = dz_to_float(io[j].e[i]);
                if (a.q_gain) {
                    const float s = kv4_square_sum<32>(x, 0xffffffffu);
                    float n = kv4_rsqrt(s * (1.0f / HD) + (float)a.eps);
                    if (!(s > 1e-25f && s < 1e37f)) {   // squares that leave fp32's range
                        double y[E];
#pragma unroll
                        for (int i = 0; i < E; i++) y[i] = (double)x[i];
                        const double m = kv4_square_sum<32>(y, 0xffffffffu) / HD + a.eps;
#pragma unroll
                        for (int i = 0; i < E; i++) x[i] = (float)(y[i] * kv4_rsqrt(m));
                        n = 1.0f;
                    }
#pragma unroll
                    for (int i = 0; i < E; i++) x[i] = gain[i] * (x[i] * n);   // x n is about 1: gains of any size
                }
                if (a.rope) kv4_rotate<HD>(x, a.halves, lane, at, [&](int i) { return angles_f[r * P + pair0 + i]; });
                kv8_store<T, E>(out + r * a.ldqo, cut.wide, x);
            }
            continue;
        }
        const bool key = item < a.c.kv_heads;
        const int h = key ? item : item - a.c.kv_heads;
        const long long ld = key ? a.ldk : a.ldv;
        const T* in = static_cast<const T*>(key ? a.k : a.v) + row0 * ld + h * HD + at;
        if (!held) continue;                 // the whole block alike
        float x[KV8_ROWS][E];
        unsigned top = 0;                    // bits of the largest magnitude; above 0x7f7fffff it is not finite
        {
            Kv8Lane<T, E> io[KV8_ROWS];
#pragma unroll
            for (int j = 0; j < KV8_ROWS; j++) {
                const int r = rank + j * team;
                if (r < rows) kv8_load<T, E>(in + r * ld, cut.wide, io[j]);
            }
#pragma unroll
            for (int j = 0; j < KV8_ROWS; j++) {
                const int r = rank + j * team;
                if (r < rows) {
#pragma unroll
                    for (int i = 0; i < E; i++) x[j][i] = dz_to_float(io[j].e[i]);
                    if (key && (a.k_gain || a.rope)) {
                        double y[E];
#pragma unroll
                        for (int i = 0; i < E; i++) y[i] = (double)x[j][i];
                        if (a.k_gain) {
                            const double n = kv4_rsqrt(kv4_square_sum<32>(y, 0xffffffffu) / HD + a.eps);
#pragma unroll
                            for (int i = 0; i < E; i++) y[i] = (double)a.k_gain[at + i] * y[i] * n;
                        }
                        if (a.rope)
                            kv4_rotate<HD>(y, a.halves, lane, at, [&](int i) { return angles[r * P + pair0 + i]; });
#pragma unroll
                        for (int i = 0; i < E; i++) x[j][i] = (float)y[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < E; i++) x[j][i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < E; i++) top = max(top, __float_as_uint(x[j][i]) & 0x7fffffffu);
            }
        }
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
        const long long place = (long long)where_page * a.c.kv_heads + h;      // the page's head
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
        const bool poisoned = top > 0x7f7fffffu || old != old;
        const float fresh = __fdiv_rn(__uint_as_float(top), 127.0f);
        const float scale = poisoned ? __int_as_float(0x7fc00000) : fmaxf(old, fresh);
        const float inverse = __fdiv_rn(1.0f, scale);
        int8_t* codes = (key ? a.c.k_codes : a.c.v_codes) + place * (a.c.page * HD);
        if (scale > old && offset) {         // the earlier rows take the larger scale
            const float ratio = __fdiv_rn(old, scale);
            for (int i = rank * 32 + lane; i < offset * (HD / 16); i += team * 32) {
                uint4* word = reinterpret_cast<uint4*>(codes) + i;
                uint4 v = *word;
                unsigned* w = reinterpret_cast<unsigned*>(&v);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    unsigned n = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int c = (int)(int8_t)(w[q] >> (8 * e));
                        n |= ((unsigned)kv8_round(__fmul_rn((float)c, ratio)) & 0xffu) << (8 * e);
                    }
                    w[q] = n;
                }
                *word = v;
            }
        }
        if (rank == 0 && lane == 0) scales[place] = scale;
        T* out = static_cast<T*>(key ? a.k_out : a.v_out);
        const long long ldo = key ? a.ldko : a.ldvo;
        if (out) out += row0 * ldo + h * HD + at;
#pragma unroll
        for (int j = 0; j < KV8_ROWS; j++) {
            const int r = rank + j * team;
            if (r >= rows) break;
            unsigned word = 0;
#pragma unroll
            for (int i = 0; i < E; i++) {
                // zeros where the scale's inverse is not finite: 0 * inf is a NaN, and rounds to 0
                const int c = poisoned || scale == 0.0f ? 0 : kv8_round(__fmul_rn(x[j][i], inverse));
                word |= ((unsigned)c & 0xffu) << (8 * i);
                x[j][i] = (float)c * scale;
            }
            int8_t* to = codes + (offset + r) * HD + at;
            if (E == 4)
                *reinterpret_cast<unsigned*>(to) = word;
            else
                *reinterpret_cast<unsigned short*>(to) = (unsigned short)word;
            if (out) kv8_store<T, E>(out + r * ldo, cut.wide, x[j]);
        }
    }
}

constexpr int KV8_DEVICES = 64;

template <typename T, int HD> static cudaError_t kv8_append_t(const Kv8AppendArgs& a, int device, int sms, cudaStream_t st) {
    static std::atomic<bool> ready[KV8_DEVICES];
    constexpr int most = 64 * (HD / 2) * (int)(sizeof(double2) + sizeof(float2));
    if (!ready[device].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(dz_kv8_append_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return e;
        ready[device].store(true, std::memory_order_release);
    }
    Kv8AppendCut cut;
    const int rows = a.n_tokens < a.c.page ? a.n_tokens : a.c.page;          // of a block at most
    cut.runs = (int)(((long long)a.n_tokens + a.c.page - 2) / a.c.page) + 1;
    for (cut.team = 1; cut.team * KV8_ROWS < rows;) cut.team *= 2;
    // four blocks to an SM, as far as there are heads for their teams
    const long long blocks = (long long)a.c.batch * cut.runs, teams = KV8_WARPS / cut.team;
    const long long heads = (2 * a.c.kv_heads + a.q_heads + teams - 1) / teams;
    long long parts = (4LL * sms + blocks - 1) / blocks;
    cut.parts = (int)(parts < heads ? parts : heads);
    constexpr int B = HD / 32 * (int)sizeof(T);
    const uintptr_t bases = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.k_out |
                            (uintptr_t)a.v_out;
    const long long strides = a.ldq | a.ldk | a.ldv | a.ldqo | a.ldko | a.ldvo;
    cut.wide = bases % B == 0 && strides * (long long)sizeof(T) % B == 0;
    cut.table_rows = a.rope ? rows : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(blocks * cut.parts));
    cfg.blockDim = dim3(KV8_WARPS * 32);
    cfg.dynamicSmemBytes = (size_t)cut.table_rows * (HD / 2) * (sizeof(double2) + sizeof(float2));
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, dz_kv8_append_kernel<T, HD>, a, cut);
}

template <typename T> static cudaError_t kv8_append_h(const Kv8AppendArgs& a, int head_dim, int device, int sms, cudaStream_t st) {
    return head_dim == 128 ? kv8_append_t<T, 128>(a, device, sms, st) : kv8_append_t<T, 64>(a, device, sms, st);
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
