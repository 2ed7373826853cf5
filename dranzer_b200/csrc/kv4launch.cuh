// How the 4-bit attention kernels (kv4attn.cu, kv4chunk.cu) are launched: units
// of work go to teams of warps or to clusters of blocks.
#pragma once
#include <atomic>

#include "kv4.cuh"

namespace dz {

constexpr int KV4_WARPS = 8;      // warps of a block
constexpr int KV4_TILE = 32;      // tokens that a warp takes at a time
constexpr int KV4_CLUSTER = 16;   // blocks of a cluster at most
constexpr int KV4_DEVICES = 64;   // devices whose launch state is kept

// Clusters of 1..16 blocks of a kernel that a device holds at once (a cluster
// stays within one GPC, so that larger ones leave SMs idle; 0: it cannot hold
// one). Asked once per kernel and device.
struct Kv4Room {
    std::atomic<bool> known{false};
    std::atomic<int> clusters[KV4_CLUSTER + 1];
};

// Warps of a team and blocks of a cluster for `units` units of up to `longest`
// visible tokens: the least number of tiles that a warp works through one
// after the other, its start (as long as 4 tiles) and the joins (3 each) among
// them. 256 x 16 units of 640 tokens: 76 us with a warp each, 123 with eight;
// 16 units of 130000: 564 us with eight, 118 with 64, 78 with 104.
inline void kv4_shape(const Kv4Room& room, long long units, long long longest, int* team, int* cluster) {
    const long long tiles = (longest + KV4_TILE - 1) / KV4_TILE;
    double best = 1e30;
    auto consider = [&](int w, int c) {
        const long long warps = (long long)w * c;
        const long long slots = (long long)room.clusters[c].load(std::memory_order_relaxed) * (KV4_WARPS / w);
        if (slots <= 0) return;
        const double waves = (double)((units + slots - 1) / slots), each = (double)((tiles + warps - 1) / warps);
        const double t = waves * (each + 4.0 + (warps > 1 ? 3.0 : 0.0) + (c > 1 ? 3.0 : 0.0));
        if (t < best) {
            best = t;
            *team = w;
            *cluster = c;
        }
    };
    for (int w = 1; w <= KV4_WARPS; w *= 2) consider(w, 1);
    for (int c = 2; c <= KV4_CLUSTER && (long long)(c - 1) * KV4_WARPS < tiles; c++) consider(KV4_WARPS, c);
}

// Enqueues kernel(a, team, cluster, blocks of pairs, units), each block with
// `smem` bytes, a unit holding `pairs_per_unit` pairs.
template <typename Kernel>
cudaError_t kv4_launch(Kernel* kernel, Kv4Room (&rooms)[KV4_DEVICES], const Kv4AttnArgs& a, int pairs_per_unit, int smem,
                       int device, cudaStream_t st) {
    if (device < 0 || device >= KV4_DEVICES) return cudaErrorInvalidDevice;
    Kv4Room& room = rooms[device];
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(KV4_WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    if (!room.known.load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        for (int c = 1; c <= KV4_CLUSTER && e == cudaSuccess; c++) {
            cfg.gridDim = dim3(c);
            attr[0].val.clusterDim.x = c;
            int n = 0;
            e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
            room.clusters[c].store(n, std::memory_order_relaxed);
        }
        if (e != cudaSuccess) return e;
        room.known.store(true, std::memory_order_release);
    }
    const int pairs = a.n_tokens * (a.q_heads / a.c.kv_heads), blocks = (pairs + pairs_per_unit - 1) / pairs_per_unit;
    const long long units = (long long)a.c.batch * a.c.kv_heads * blocks, ring = a.c.capacity - a.c.sinks;
    const long long longest = a.c.sinks + (a.window && a.window < ring ? a.window + a.n_tokens : ring);
    int team = 1, cluster = 1;
    kv4_shape(room, units, longest, &team, &cluster);
    cfg.gridDim = dim3((unsigned)((units + KV4_WARPS / team - 1) / (KV4_WARPS / team) * cluster));
    attr[0].val.clusterDim.x = cluster;
    cfg.attrs = cluster > 1 ? attr : attr + 1;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, team, cluster, blocks, (int)units);
}

}  // namespace dz
