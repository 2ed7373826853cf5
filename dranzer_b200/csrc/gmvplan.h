// How a group-scaled product (gmatvec.cu) is cut: the shared memory of a block
// and the choice of rows, clusters and tiles. Host arithmetic alone, without a
// CUDA header.
#pragma once
#include <atomic>

#ifdef __CUDACC__
#define DZ_HD __host__ __device__
#else
#define DZ_HD
#endif

namespace dz {

constexpr int GMV_TILE = 32;     // columns of a tile
constexpr int GMV_BLOCK = 128;   // rows of a block
constexpr int GMV_CODES = GMV_TILE * GMV_BLOCK / 2;

constexpr int GMV_SMEM = 227 * 1024 - 128;// shared memory a block may have
constexpr int GMV_SMEM2 = 113 * 1024 - 128;// and if two are to fit an SM
constexpr int GMV_WARPS = 8;
constexpr int GMV_STAGES = 4;
constexpr int GMV_MAX_ROWS = 16;        // rows of one pass
constexpr int GMV_DIGITS = 8;           // of an activation of a single row

struct GmvPlan {
    int rows;         // rows of this launch
    int digits;       // whether its one row goes as digits
    int cluster;      // blocks that share a tile
    int clusters;     // clusters of the grid
    int slice;        // records of a tile that a block has, at most
    int tiles;        // tiles of a cluster, at most
};

// Shared memory: the rings, the columns of activations (or digits and their
// weights), a warp's tile in accumulator order, the parts.
template <int P, int NT> struct GmvSmem {   // NT 0: one row as digits
    static constexpr int TILES = NT ? NT : 1;
    static constexpr int LD = 8 * TILES + 1;                 // floats between the columns of W in a warp's tile
    static constexpr int TILE = (GMV_TILE * LD + 3) / 4 * 4;
    static DZ_HD int ring(int rec) { return GMV_WARPS * GMV_STAGES * rec; }
    // bytes between columns: what neighbours read of a piece (64 bytes, 32 of digits) falls into different banks
    static DZ_HD int stride(int slice) { return NT ? slice * GMV_BLOCK * 2 + 64 : slice * GMV_BLOCK + 32; }
    static DZ_HD int columns(int rows, int slice) {
        return NT ? P * rows * stride(slice) : GMV_DIGITS * stride(slice) + slice * GMV_DIGITS * 4;
    }
    static DZ_HD int total(int rec, const GmvPlan& p) {
        return ring(rec) + columns(p.rows, p.slice) + GMV_WARPS * TILE * 4 + (p.tiles + GMV_WARPS) * GMV_TILE * p.rows * 4;
    }
};

// Blocks of an instantiation that an SM is to hold: its registers would not let
// more tiles or groups share it without spills.
constexpr int gmv_blocks(int nt, int gpb) { return nt < 3 || (nt == 3 && gpb == 1) ? 2 : 1; }

// What the cut depends on: a matrix's tiles, blocks and records, the columns of B
// that an activation takes (3 of fp32, else 1).
struct GmvShape {
    int ntiles, nblocks, group, rec_bytes, parts;
};

// Column tiles of 8 for `rows` rows: the instantiations of the kernel.
inline int gmv_col_tiles(int parts, int rows) {
    const int n = (parts * rows + 7) / 8;
    return n <= 3 ? n : 6;
}

inline int gmv_smem(const GmvShape& a, const GmvPlan& p) {
    const int nt = gmv_col_tiles(a.parts, p.rows), rec = a.rec_bytes;
    if (p.digits) return GmvSmem<1, 0>::total(rec, p);
    if (a.parts == 3)
        return nt == 1   ? GmvSmem<3, 1>::total(rec, p)
               : nt == 2 ? GmvSmem<3, 2>::total(rec, p)
               : nt == 3 ? GmvSmem<3, 3>::total(rec, p)
                         : GmvSmem<3, 6>::total(rec, p);
    return nt == 1 ? GmvSmem<1, 1>::total(rec, p) : GmvSmem<1, 2>::total(rec, p);
}

// Clusters of 1, 2, 4, 8 and 16 blocks that `device` holds at once with one
// block on an SM, then with two (a cluster stays within one GPC, so that larger
// ones leave SMs idle; 0: it cannot hold one). Asked once per device.
struct GmvRoom {
    std::atomic<bool> known{false};
    std::atomic<int> clusters[2][5];
};

// How a tile is shared: the shape with the least estimated time. False: none that
// the device can hold takes the rows' activations. The estimate, in us on one B200 (K 256..12032, N
// 48..32000, 1..16 rows): four loads of activations by every thread 0.9 (16 bits:
// 0.6), from the third time on 0.6 more, whose latency nothing hides; a record
// 0.38 when all SMs stream from HBM, and by its own latency 0.3 + 0.15 NT + 0.02
// NT GPB; a cluster's join 1.0, 0.16 per block and what each reads of the others.
// 16 x 4096 x 4096 in fp32: 33 us with one block to a tile, 20 with two, 17 with
// four, 14 with eight; 2 x 4096 x 4096: 5.8, 6.2, 6.2 and 6.7 us.
inline bool gmv_plan_as(const GmvShape& a, int rows, int digits, const GmvRoom& room, GmvPlan* plan) {
    const int gpb = GMV_BLOCK / a.group, nt = digits ? 0 : gmv_col_tiles(a.parts, rows);
    double cost = 1e30;
    for (int i = 0; i < 5 && (1 << i) <= a.nblocks; i++) {
        if (i == 4 && cost < 1e30) break;              // 16 blocks only where 8 cannot hold their rows' activations
        for (int two = 0; two < gmv_blocks(nt, gpb); two++) {
            GmvPlan p;
            const int c = 1 << i, fits = room.clusters[two][i].load(std::memory_order_relaxed);
            if (fits <= 0) continue;
            p.rows = rows;
            p.digits = digits;
            p.cluster = c;
            p.slice = (a.nblocks + c - 1) / c;
            p.clusters = fits < a.ntiles ? fits : a.ntiles;
            p.tiles = (a.ntiles + p.clusters - 1) / p.clusters;
            if (gmv_smem(a, p) > (two ? GMV_SMEM2 : GMV_SMEM)) continue;
            const int per_batch = GMV_WARPS * (a.parts == 3 ? 4 : 8), batches = (rows * p.slice + per_batch - 1) / per_batch;
            const double stage = (a.parts == 3 ? 0.9 : 0.6) * batches + 0.6 * (batches > 2 ? batches - 2 : 0);
            const double stream = 0.38 * (two + 1), own = (0.3 + 0.15 * nt + 0.02 * nt * gpb) * (two ? 1.6 : 1.0);
            const double t = stage * (two ? 1.6 : 1.0) +
                             (stream > own ? stream : own) * ((p.tiles * p.slice + GMV_WARPS - 1) / GMV_WARPS) +
                             (c > 1 ? 1.0 + 0.16 * c + 0.0125 * p.tiles * rows : 0.0);
            if (t < cost) {
                cost = t;
                *plan = p;
            }
        }
    }
    return cost < 1e30;
}

// How many rows a pass takes, and how: half as many where no shape holds them.
inline bool gmv_plan(const GmvShape& a, int rows, const GmvRoom& room, GmvPlan* plan) {
    if (rows == 1 && gmv_plan_as(a, 1, 1, room, plan)) return true;
    for (rows = rows < GMV_MAX_ROWS ? rows : GMV_MAX_ROWS; rows >= 1; rows /= 2)
        if (gmv_plan_as(a, rows, 0, room, plan)) return true;
    return false;
}

// The tiles that one launch takes of the matrix's last `tiles` (their sums lie in
// shared memory), and its plan; 0: not even one.
inline int gmv_plan_tiles(const GmvShape& a, int tiles, int rows, const GmvRoom& room, GmvPlan* plan) {
    GmvShape s = a;
    for (s.ntiles = tiles; s.ntiles >= 1; s.ntiles /= 2)
        if (gmv_plan(s, rows, room, plan)) return s.ntiles;
    return 0;
}

}  // namespace dz
