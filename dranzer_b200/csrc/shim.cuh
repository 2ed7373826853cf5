// What every translation unit with C entry points shares: the calling
// thread's last error, the device switch of a call, and the activation types
// of the 4-bit operators (dz_types.h, DZ_TYPE_*).
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "dz_types.h"

namespace dz {

// Records `status` and the message for dz_cuda_last_error; returns `status`.
int fail(int status, const char* fmt, ...);

#define DZ_CUDA(call)                                                                      \
    do {                                                                                   \
        cudaError_t e_ = (call);                                                           \
        if (e_ != cudaSuccess) {                                                           \
            (void)cudaGetLastError(); /* not left for a later call to find */              \
            return fail(e_ == cudaErrorMemoryAllocation ? DZ_E_NOMEM : DZ_E_DEVICE,        \
                        "%s: %s (%s:%d)", #call, cudaGetErrorString(e_), __FILE__, __LINE__); \
        }                                                                                  \
    } while (0)

// Switches to a handle's device for the duration of a call.
struct DeviceGuard {
    int prev = -1;
    bool ok = true;
    explicit DeviceGuard(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev != dev) ok = cudaSetDevice(dev) == cudaSuccess;
    }
    ~DeviceGuard() {
        int cur;
        if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
    }
};

inline bool type_ok(int type) { return type == DZ_TYPE_F32 || type == DZ_TYPE_F16 || type == DZ_TYPE_BF16; }
inline size_t type_bytes(int type) { return type == DZ_TYPE_F32 ? 4 : 2; }

// One element of a typed activation array: exact widening, one rounding back.
template <typename T> __device__ __forceinline__ float dz_to_float(T v);
template <> __device__ __forceinline__ float dz_to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float dz_to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float dz_to_float<__nv_bfloat16>(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
template <typename T> __device__ __forceinline__ T dz_from_float(float v);
template <> __device__ __forceinline__ float dz_from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half dz_from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 dz_from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

}  // namespace dz
