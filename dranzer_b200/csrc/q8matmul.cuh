// What the kernels of the 8-bit products share (q8matmul.cu: few rows,
// q8gemm.cu: the tensor cores of the 5th generation).
#pragma once
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

#include "q8plan.h"
#include "shim.cuh"

namespace dz {

constexpr int Q8_DEVICES = 64;     // devices whose launch state is kept

struct Q8MatArgs {
    const int8_t* a;
    long long lda;
    const float* a_scales;
    const int8_t* levels;
    const float* col_scale;
    const float* bias;
    void* c;
    long long ldc;
    int M, N, K, nkb;
};

template <typename T> __device__ __forceinline__ T q8_finish(int sum, float a_scale, float col_scale, float bias) {
    return dz_from_float<T>(fmaf((float)sum * a_scale, col_scale, bias));
}

// The product on the tensor cores, in tiles of 32 rows and more; `levels` maps
// the matrix's level blocks.
[[nodiscard]] cudaError_t dz_q8gemm_launch(const Q8MatArgs& a, const CUtensorMap& levels, const Q8Plan& plan, int type,
                                           int device, int sms, cudaStream_t st);

}  // namespace dz
