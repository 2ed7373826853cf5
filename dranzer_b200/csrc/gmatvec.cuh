// Products with group-scaled 4-bit weights: y[m][n] = sum_g s[g][n] *
// sum_{k in g} (c[k][n] - 7) x[m][k], groups of 32, 64 or 128 rows.
//
// Device layout. The matrix is cut into tiles of 32 columns and blocks of 128
// rows; one (tile, block) is one record, tile major: 2 KB of codes, then the
// block's scales [128 / group][32] (fp32 or fp16). The codes are four pieces
// of 512 B, one for each 32 rows. In a piece, lane l = 4g + t of a warp owns 16
// bytes, four words: columns g, g + 8, g + 16 and g + 24 at rows 8t..8t+7 of
// the piece. A word holds eight levels (code - 7) as two's complement nibbles:
// byte j has row 8t + j in its high half and row 8t + 4 + j in its low half, so
// that one AND (high) or one shift and one AND (low) leaves 16 x level in four
// signed bytes: a fragment register of the 8-bit integer MMA (m16n8k32, rows
// = columns of W). Rows past K and columns past N hold level 0 and scale 0.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "gmvplan.h"

namespace dz {

struct GmvMatrix {
    uint8_t* rec = nullptr;      // [ntiles][nblocks] records
    int K = 0, N = 0, group = 0;
    int scale_f16 = 0;
    int ntiles = 0, nblocks = 0;
    int rec_bytes = 0;
};

struct GmvArgs {
    GmvMatrix w;
    const void* x;
    void* y;
    long long ldx, ldy;
    int M;
    int type;                    // DZ_TYPE_* of x and y
};

// Enqueues the product of any number of rows.
cudaError_t dz_gmv_launch(const GmvArgs& a, int device, cudaStream_t st);

}  // namespace dz
