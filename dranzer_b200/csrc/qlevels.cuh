// The level blocks of a quantized matrix handle, for products outside dz_cuda.cu.
#pragma once
#include <cstdint>
#include <cuda.h>

#include "dz_cuda.h"

namespace dz {

struct QLevels {
    int device, K, N, gran;
    const int8_t* levels;      // [n / 128][k / 128][n % 128][k % 128], zero past K and N; null: none kept
    const float* col_scale;    // [N rounded up to 16]
    CUtensorMap map;           // of `levels`: boxes of 128 k x 128 n, 128-byte swizzle
};
void dz_qmatrix_levels(const dz_cuda_qmatrix_t* matrix, QLevels* out);

// A tiled uint8 TMA map with the 64- or 128-byte swizzle (as wide as box[0])
// over a tensor of `rank` dims (dims[0] innermost, strides in bytes for dims 1..).
bool dz_encode_u8_map(CUtensorMap* tm, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                      const uint32_t* box);

}  // namespace dz
