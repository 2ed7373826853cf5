// The norm and the rotation of a head that the lanes of a warp share, for the
// appends to 4-bit and 8-bit caches.
#pragma once
#include <cuda_runtime.h>

namespace dz {

template <int LANES> __device__ __forceinline__ unsigned kv4_mask(int lane) {   // the lanes of a group of LANES
    return LANES == 32 ? 0xffffffffu : ((1u << (LANES & 31)) - 1u) << (lane & ~(LANES - 1));
}

// 1 / sqrt(m): the approximation and Newton's step r (3 - m r^2) / 2, once in
// fp32 (to about 2^-23) and twice in 64 bits (2^-22 squares to 2^-43, 2^-85);
// the functions where m leaves fp32's range.
__device__ __forceinline__ float kv4_rsqrt(float m) {
    const float r = rsqrtf(m);
    return r * fmaf(-0.5f * m * r, r, 1.5f);
}
__device__ __forceinline__ double kv4_rsqrt(double m) {
    if (!(m > 1e-30 && m < 1e30)) return 1.0 / sqrt(m);
    double r = (double)rsqrtf((float)m);
    r = r * fma(-0.5 * m * r, r, 1.5);
    return r * fma(-0.5 * m * r, r, 1.5);
}

// Sum over the head's lanes of x^2.
template <int LPH, int E, typename A> __device__ __forceinline__ A kv4_square_sum(const A (&x)[E], unsigned mask) {
    A s = 0;
#pragma unroll
    for (int i = 0; i < E; i++) s += x[i] * x[i];
#pragma unroll
    for (int off = LPH / 2; off >= 1; off >>= 1) s += __shfl_xor_sync(mask, s, off);
    return s;
}

__device__ __forceinline__ float kv4_signed(float v, bool minus) {
    return __uint_as_float(__float_as_uint(v) ^ (minus ? 0x80000000u : 0u));
}
__device__ __forceinline__ double kv4_signed(double v, bool minus) {
    return __hiloint2double(__double2hiint(v) ^ (minus ? (int)0x80000000 : 0), __double2loint(v));
}

// Rotates a head's E elements of this lane, element `at` first; angle(i) gives
// cosine and sine of the lane's i-th pair.
template <int HD, int E, typename A, typename F>
__device__ __forceinline__ void kv4_rotate(A (&x)[E], bool halves, int lane, int at, F angle) {
    constexpr int LPH = HD / E;
    if (halves) {
        // element e pairs with e + HD / 2, which the lane half a head away holds at the same index:
        // x cos - other sin in the first half, x cos + other sin in the second
        const unsigned mask = kv4_mask<LPH>(lane);
#pragma unroll
        for (int i = 0; i < E; i++) {
            const auto q = angle(i);
            const A other = kv4_signed(__shfl_xor_sync(mask, x[i], LPH / 2), at < HD / 2);
            x[i] = x[i] * (A)q.x + other * (A)q.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            const auto q = angle(i / 2);
            const A u = x[i], v = x[i + 1];
            x[i] = u * (A)q.x - v * (A)q.y;
            x[i + 1] = u * (A)q.y + v * (A)q.x;
        }
    }
}

}  // namespace dz
