// The norm of a head that the lanes of a warp share, for the appends to 4-bit
// and 8-bit caches.
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

}  // namespace dz
