// Products of 8-bit rows with a quantized matrix on the tensor cores
// (q8matmul.cuh): D[n][m] = sum_k level[n][k] a[m][k] in kind::i8 MMAs, the
// matrix's columns as the 128 lanes of tensor memory and the rows as its
// columns, so that an output row is written by the lanes of a warp side by
// side. Both operands are K-major and come by TMA with the 128-byte swizzle,
// what lies past the rows or past k as zeros.
#include <atomic>
#include <cooperative_groups.h>

#include "q8matmul.cuh"
#include "qlevels.cuh"
#include "tcgen05.cuh"

namespace dz {

namespace cg = cooperative_groups;

constexpr int Q8G_THREADS = 256;
constexpr uint32_t Q8G_A_BYTES = 128 * 128;      // levels of a stage

constexpr int Q8G_STAGES = 10;                   // of a block at most
template <int TN> struct Q8gShape {
    static constexpr uint32_t B_BYTES = TN * 128;
    static constexpr uint32_t STAGE = Q8G_A_BYTES + B_BYTES;
    // a block alone on its SM, or one of two
    static constexpr int ALONE = (int)(200 * 1024 / STAGE), SHARED = (int)(100 * 1024 / STAGE);
    static_assert(ALONE <= Q8G_STAGES && 2 * STAGE >= TN * 128 * 4, "barriers of a stage; parts' sums in two stages");
    static constexpr size_t smem(int stages) { return (size_t)stages * STAGE + 1024 + 256; }
};

// kind::i8, int32 sums, both operands s8 and K-major, 128 lanes, TN columns.
template <int TN> __device__ __forceinline__ uint32_t q8g_idesc() {
    return 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(TN >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
}

__device__ __forceinline__ void q8g_tma_2d(void* dst, const CUtensorMap* tm, int c0, int c1, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dz_smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(c1), "r"(dz_smem_addr(bar))
        : "memory");
}

// A block takes 128 columns, TN rows and a share of k; the blocks of a cluster
// split k and add their sums through distributed shared memory.
template <typename T, int TN>
__global__ void __launch_bounds__(Q8G_THREADS, 2)
    dz_q8gemm_kernel(const __grid_constant__ CUtensorMap tm_levels, const __grid_constant__ CUtensorMap tm_rows,
                     const __grid_constant__ Q8MatArgs a, int stages, int mtiles, int parts) {
    using S = Q8gShape<TN>;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(1024) uint8_t q8g_raw[];
    uint8_t* sm = q8g_raw + ((1024u - (dz_smem_addr(q8g_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + (size_t)stages * S::STAGE);
    uint64_t* empty = full + Q8G_STAGES;
    uint64_t* accum = empty + Q8G_STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accum + 1);
    int* progress = reinterpret_cast<int*>(tmem_slot + 1);       // stages issued, consumed; failed
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // parts of a tile side by side, then the tiles of the same levels
    const int part = (int)(blockIdx.x % (unsigned)parts), where = (int)(blockIdx.x / (unsigned)parts);
    const int tile = where / mtiles, n0 = tile * 128, m0 = where % mtiles * TN;
    const int kb0 = (int)((long long)a.nkb * part / parts), nkb = (int)((long long)a.nkb * (part + 1) / parts) - kb0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; s++) {
            dz_mbar_init(&full[s]);
            dz_mbar_init(&empty[s]);
        }
        dz_mbar_init(accum);
        progress[0] = progress[1] = progress[2] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dz_smem_addr(tmem_slot)),
                     "r"((uint32_t)TN)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    ug_fence_before();
    __syncthreads();
    ug_fence_after();
    const uint32_t tmem = *tmem_slot;
    if (warp == 0) {
        const bool elected = ug_elect();
        // the levels of the first stages are no kernel's output and go out before the one before has ended
        const int pre = nkb < stages ? nkb : stages;
        for (int kb = 0; kb < pre; kb++)
            if (elected) {
                dz_mbar_expect_tx(&full[kb], S::STAGE);
                ug_tma_4d(sm + (size_t)kb * S::STAGE, &tm_levels, 0, 0, kb0 + kb, tile, &full[kb]);
            }
        asm volatile("griddepcontrol.wait;" ::: "memory");
        int kb = 0, s = 0;
        uint32_t phase = 1;                  // of the stage's consumption before
        for (; kb < nkb; kb++) {
            if (kb >= stages && !dz_mbar_wait(&empty[s], phase)) {
                if (elected) progress[2] = 1;
                break;
            }
            uint8_t* to = sm + (size_t)s * S::STAGE;
            if (elected) {
                if (kb >= pre) {
                    dz_mbar_expect_tx(&full[s], S::STAGE);
                    ug_tma_4d(to, &tm_levels, 0, 0, kb0 + kb, tile, &full[s]);
                }
                q8g_tma_2d(to + Q8G_A_BYTES, &tm_rows, (kb0 + kb) * 128, m0, &full[s]);
            }
            if (++s == stages) {
                s = 0;
                phase ^= 1;
            }
        }
        if (elected) progress[0] = kb;
        __syncwarp();
    } else if (warp == 1) {
        // barrier waits are bounded, the kernel before is not: none begins before it has ended
        asm volatile("griddepcontrol.wait;" ::: "memory");
        const bool elected = ug_elect();
        const uint64_t first = ug_desc_kmajor(dz_smem_addr(sm));
        int kb = 0, s = 0;
        uint32_t phase = 0;
        for (; kb < nkb; kb++) {
            if (!dz_mbar_wait(&full[s], phase)) {
                if (elected) progress[2] = 1;
                break;
            }
            ug_fence_after();
            const uint64_t levels = first + (uint64_t)(s * (S::STAGE >> 4)), rows = levels + (Q8G_A_BYTES >> 4);
            if (elected) {
#pragma unroll
                for (int kk = 0; kk < 4; kk++)
                    ug_mma(tmem, levels + kk * 2, rows + kk * 2, q8g_idesc<TN>(), (kb > 0 || kk > 0) ? 1u : 0u);
                ug_commit(&empty[s]);
            }
            __syncwarp();
            if (++s == stages) {
                s = 0;
                phase ^= 1;
            }
        }
        if (elected) {
            progress[1] = kb;
            ug_commit(accum);
        }
        __syncwarp();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the rows' scales; and the waits above
    const bool ok = dz_mbar_wait(accum, 0);
    ug_fence_after();
    const bool failed = !ok || progress[2];
    T* c = static_cast<T*>(a.c);
    const T nothing = dz_from_float<T>(__int_as_float(0x7fc00000));
    if (parts == 1) {
        // a thread has a column, half of the warps the first rows
        const int n = n0 + (warp & 3) * 32 + lane;
        const float scale = n < a.N ? a.col_scale[n] : 0.0f, bias = n < a.N && a.bias ? a.bias[n] : 0.0f;
        for (int c0 = (warp >> 2) * 32; c0 < TN && m0 + c0 < a.M; c0 += 64) {
            int32_t v[32];
            ug_tmem_ld32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c0, v);
            if (n < a.N) {
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    const int m = m0 + c0 + i;
                    if (m < a.M) c[m * a.ldc + n] = failed ? nothing : q8_finish<T>(v[i], a.a_scales[m], scale, bias);
                }
            }
        }
    } else {
        // sums to shared memory (the stages' place, all consumed), [row][column], and the cluster's parts of a row added
        int* sums = reinterpret_cast<int*>(sm);
        for (int c0 = (warp >> 2) * 32; c0 < TN; c0 += 64) {
            int32_t v[32];
            ug_tmem_ld32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c0, v);
#pragma unroll
            for (int i = 0; i < 32; i++) sums[(c0 + i) * 128 + (warp & 3) * 32 + lane] = v[i];
        }
        int* any = progress + 2;
        if (failed && lane == 0) *any = 1;
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const int rows = min(TN, a.M - m0);
        const int first = rows * part / parts, last = rows * (part + 1) / parts;
        bool lost = false;
        for (int p = 0; p < parts; p++) lost |= *cluster.map_shared_rank(any, p) != 0;
        // a warp has a row, a lane four of its columns, all parts' sums in flight together
        const int n = n0 + 4 * lane;
        float scale[4], bias[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            scale[e] = n + e < a.N ? a.col_scale[n + e] : 0.0f;
            bias[e] = n + e < a.N && a.bias ? a.bias[n + e] : 0.0f;
        }
        const int* from[Q8_PARTS];
#pragma unroll
        for (int p = 0; p < Q8_PARTS; p++) from[p] = cluster.map_shared_rank(sums, p < parts ? p : part) + 4 * lane;
#pragma unroll 2
        for (int r = first + warp; r < last; r += Q8G_THREADS / 32) {
            int4 v[Q8_PARTS];
#pragma unroll
            for (int p = 0; p < Q8_PARTS; p++)
                v[p] = p < parts ? *reinterpret_cast<const int4*>(from[p] + r * 128) : make_int4(0, 0, 0, 0);
            const float row = a.a_scales[m0 + r];
            int sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < Q8_PARTS; p++) {
                sum[0] += v[p].x;
                sum[1] += v[p].y;
                sum[2] += v[p].z;
                sum[3] += v[p].w;
            }
            T* to = c + (long long)(m0 + r) * a.ldc + n;
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (n + e < a.N) to[e] = lost ? nothing : q8_finish<T>(sum[e], row, scale[e], bias[e]);
        }
        cluster.sync();                      // no block ends while another reads its shared memory
    }
    // copies and MMAs in flight end before the shared memory and the tensor memory are released
    ug_fence_before();
    if (threadIdx.x == 0 && progress[2]) {
        for (int kb = progress[1]; kb < progress[0]; kb++)
            if (!dz_mbar_wait(&full[kb % stages], (uint32_t)((kb / stages) & 1))) break;
        dz_mbar_wait(accum, 0);
    }
    __syncthreads();
    if (warp == 1) {
        ug_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)TN) : "memory");
    }
}

template <typename T, int TN>
static cudaError_t q8gemm_t(const Q8MatArgs& a, const CUtensorMap& levels, int parts, int device, int sms, cudaStream_t st) {
    static std::atomic<bool> ready[Q8_DEVICES];
    using S = Q8gShape<TN>;
    const auto kernel = dz_q8gemm_kernel<T, TN>;
    if (!ready[device].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::smem(S::ALONE));
        if (e != cudaSuccess) return e;
        ready[device].store(true, std::memory_order_release);
    }
    CUtensorMap rows;
    const uint64_t dims[2] = {(uint64_t)a.K, (uint64_t)a.M}, strides[1] = {(uint64_t)a.lda};
    const uint32_t box[2] = {128, (uint32_t)TN};
    if (!dz_encode_u8_map(&rows, a.a, 2, dims, strides, box)) return cudaErrorInvalidValue;
    const int tiles = (a.N + 127) / 128, mtiles = (a.M + TN - 1) / TN;
    const long long blocks = (long long)tiles * mtiles * parts;
    // no more stages than a block has steps: clusters of blocks that fill an SM each find few places
    const int most = blocks <= sms ? S::ALONE : S::SHARED, steps = (a.nkb + parts - 1) / parts;
    const int stages = steps >= most ? most : steps < 2 ? 2 : steps;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(Q8G_THREADS);
    cfg.dynamicSmemBytes = S::smem(stages);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, levels, rows, a, stages, mtiles, parts);
}

// ------------------------------------------------- many rows: pairs of SMs
//
// Two blocks of a cluster share a tile of 256 columns x 256 rows
// (cta_group::2): each loads 128 columns of levels and half of the rows, 32 KB
// for 256 x 128 x 128 products of its own, where a block alone would load 48.
// The pairs stay and take tiles in turn. Two accumulators fill the tensor
// memory, so that eight warps of each block write a tile while the next one's
// MMAs run. The first block of a pair issues the MMAs for both; its `full`
// barriers count both blocks' bytes, commits arrive at both blocks' barriers.

constexpr int Q8P_WRITERS = 8;
constexpr int Q8P_THREADS = 64 + Q8P_WRITERS * 32;   // warp 0 copies, warp 1 MMAs, the others outputs
constexpr int Q8P_TILE = 256;
constexpr uint32_t Q8P_STAGE = 2 * 128 * 128;
constexpr int Q8P_STAGES = 6;
constexpr size_t Q8P_SMEM = (size_t)Q8P_STAGES * Q8P_STAGE + 1024 + 256 + 2 * Q8P_TILE * sizeof(float);
// A block of the next kernel may arrive before those of this one have their
// tensor memory, and keeps its own until this kernel has ended. So no two blocks
// that an SM holds at once may want more than 512 columns: a pair's block and
// any other of a product exceed the shared memory, dz_q8gemm_kernel's two (by
// their registers) have 128 columns each at most.
static_assert(Q8P_SMEM + Q8gShape<32>::smem(2) > 227 * 1024, "blocks beside one of a pair");
constexpr int Q8P_BAND = 8;                      // tiles of rows that neighbouring pairs share columns over

__device__ __forceinline__ uint32_t q8p_at_leader(const void* p) {       // the same place in the pair's first block
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(dz_smem_addr(p)));
    return r;
}
__device__ __forceinline__ void q8p_tma_4d(void* dst, const CUtensorMap* tm, int c2, int c3, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %3, %4}], "
        "[%5];" ::"r"(dz_smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(0), "r"(c2), "r"(c3), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void q8p_tma_2d(void* dst, const CUtensorMap* tm, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dz_smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void q8p_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate) {
    const uint32_t idesc = 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(256 >> 3) << 17 | (uint32_t)(256 >> 4) << 24;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives at `bar` of both blocks once every MMA issued so far has completed.
__device__ __forceinline__ void q8p_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                     dz_smem_addr(bar)),
                 "h"((unsigned short)3)
                 : "memory");
}
// dz_mbar_wait for barriers that the other block arrives at.
__device__ __forceinline__ bool q8p_test(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(dz_smem_addr(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ bool q8p_wait(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
    for (int i = 0; i < 4; i++)
        if (q8p_test(bar, parity)) return true;
    const uint64_t t0 = dz_global_ns();
    for (unsigned i = 0;; i++) {
        if (q8p_test(bar, parity)) return true;
        if ((i & 255u) == 255u && dz_global_ns() - t0 > 1000000000ull) return false;
    }
}

// Tile i of the grid: bands of Q8P_BAND tiles of rows, columns in turn within a
// band, so that the pairs at work at a time share both operands in L2.
__device__ __forceinline__ void q8p_place(int i, int ntiles, int mtiles, int* n, int* m) {
    const int band = i / (Q8P_BAND * ntiles), within = i - band * Q8P_BAND * ntiles;
    const int high = min(Q8P_BAND, mtiles - band * Q8P_BAND);
    *n = within / high;
    *m = band * Q8P_BAND + within % high;
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Q8P_THREADS, 1)
    dz_q8pair_kernel(const __grid_constant__ CUtensorMap tm_levels, const __grid_constant__ CUtensorMap tm_rows,
                     const __grid_constant__ Q8MatArgs a, int ntiles, int mtiles) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(1024) uint8_t q8g_raw[];
    uint8_t* sm = q8g_raw + ((1024u - (dz_smem_addr(q8g_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + (size_t)Q8P_STAGES * Q8P_STAGE);   // used in the first block
    uint64_t* empty = full + Q8P_STAGES;
    uint64_t* done = empty + Q8P_STAGES;         // [2] an accumulator is complete
    uint64_t* drained = done + 2;                // [2] and has been read by both blocks; used in the first block
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 2);
    volatile int* failed = reinterpret_cast<int*>(tmem_slot + 1);
    int* issued = reinterpret_cast<int*>(tmem_slot + 2);         // stages copied, consumed
    float* scales = reinterpret_cast<float*>(sm + (size_t)Q8P_STAGES * Q8P_STAGE + 256);   // [2][256] of the rows
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)(blockIdx.x & 1u), pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1);
    const int tiles = ntiles * mtiles;
    if (threadIdx.x == 0) {
        for (int s = 0; s < Q8P_STAGES; s++) {
            dz_mbar_init(&full[s]);
            dz_mbar_init(&empty[s]);
        }
        for (int i = 0; i < 2; i++) {
            dz_mbar_init(&done[i]);
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(dz_smem_addr(&drained[i])), "r"(2 * Q8P_WRITERS)
                         : "memory");            // their writers
        }
        *failed = 0;
        issued[0] = issued[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dz_smem_addr(tmem_slot)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    ug_fence_before();
    __syncthreads();
    cg::this_cluster().sync();                   // both blocks' barriers are ready
    ug_fence_after();
    const uint32_t tmem = *tmem_slot;
    if (warp == 0) {
        const bool elected = ug_elect();
        int step = 0, s = 0;                     // stages since the start; the next one's place
        uint32_t phase = 1;
        bool ok = true;
        for (int i = pair; i < tiles && ok; i += pairs) {
            int tn, tm;
            q8p_place(i, ntiles, mtiles, &tn, &tm);
            for (int kb = 0; kb < a.nkb; kb++, step++) {
                if (step >= Q8P_STAGES && !q8p_wait(&empty[s], phase)) {
                    ok = false;
                    break;
                }
                uint8_t* to = sm + (size_t)s * Q8P_STAGE;
                const uint32_t bar = q8p_at_leader(&full[s]);
                if (elected) {
                    if (rank == 0) dz_mbar_expect_tx(&full[s], 2 * Q8P_STAGE);
                    q8p_tma_4d(to, &tm_levels, kb, tn * 2 + rank, bar);
                }
                // the levels are no kernel's output, the rows are
                if (step == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
                if (elected) q8p_tma_2d(to + Q8G_A_BYTES, &tm_rows, kb * 128, tm * Q8P_TILE + rank * 128, bar);
                if (++s == Q8P_STAGES) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
        if (elected) {
            if (!ok) *failed = 1;
            issued[0] = step;
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            asm volatile("griddepcontrol.wait;" ::: "memory");   // before the bounded waits, as in dz_q8gemm_kernel
            const bool elected = ug_elect();
            const uint64_t first = ug_desc_kmajor(dz_smem_addr(sm));
            int step = 0, turn = 0, s = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int i = pair; i < tiles && ok; i += pairs, turn++) {
                const int b = turn & 1;
                if (turn >= 2 && !q8p_wait(&drained[b], (uint32_t)((turn / 2 - 1) & 1))) {
                    ok = false;
                    break;
                }
                ug_fence_after();
                for (int kb = 0; kb < a.nkb; kb++, step++) {
                    if (!q8p_wait(&full[s], phase)) {
                        ok = false;
                        break;
                    }
                    ug_fence_after();
                    const uint64_t levels = first + (uint64_t)(s * (Q8P_STAGE >> 4)), rows = levels + (Q8G_A_BYTES >> 4);
                    if (elected) {
#pragma unroll
                        for (int kk = 0; kk < 4; kk++)
                            q8p_mma(tmem + (uint32_t)(b * 256), levels + kk * 2, rows + kk * 2, (kb > 0 || kk > 0) ? 1u : 0u);
                        q8p_commit(&empty[s]);
                    }
                    __syncwarp();
                    if (++s == Q8P_STAGES) {
                        s = 0;
                        phase ^= 1;
                    }
                }
                if (ok && elected) q8p_commit(&done[b]);
            }
            if (elected) {
                if (!ok) *failed = 1;
                issued[1] = step;
            }
        }
        __syncwarp();
    } else {
        asm volatile("griddepcontrol.wait;" ::: "memory");   // the rows' scales
        // a warp reads the lanes of its number modulo 4: 32 columns, and half of the rows
        const int quarter = warp & 3, half = (warp - 2) / 4 * (Q8P_TILE / 2), thread = (int)threadIdx.x - 64;
        const T nothing = dz_from_float<T>(__int_as_float(0x7fc00000));
        int turn = 0;
        bool ok = true;
        for (int i = pair; i < tiles; i += pairs, turn++) {
            const int b = turn & 1;
            int tn, tm;
            q8p_place(i, ntiles, mtiles, &tn, &tm);
            const int n = tn * Q8P_TILE + rank * 128 + quarter * 32 + lane, m0 = tm * Q8P_TILE;
            const float scale = n < a.N ? a.col_scale[n] : 0.0f, bias = n < a.N && a.bias ? a.bias[n] : 0.0f;
            float* row_scales = scales + b * Q8P_TILE;
            row_scales[thread] = m0 + thread < a.M ? a.a_scales[m0 + thread] : 0.0f;
            asm volatile("bar.sync 1, %0;" ::"n"(Q8P_WRITERS * 32) : "memory");
            if (ok && !q8p_wait(&done[b], (uint32_t)((turn / 2) & 1))) {
                ok = false;                      // this tile and those after it read NaN
                *failed = 1;
            }
            ug_fence_after();
            for (int c0 = half; c0 < half + Q8P_TILE / 2 && m0 + c0 < a.M; c0 += 32) {
                int32_t v[32];
                ug_tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * 256 + c0), v);
                T* to = static_cast<T*>(a.c) + (long long)(m0 + c0) * a.ldc + n;
                const int rows = min(32, a.M - m0 - c0);
                if (n < a.N) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 r = *reinterpret_cast<const float4*>(row_scales + c0 + j);
                        const float y[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            if (j + e < rows) *to = ok ? q8_finish<T>(v[j + e], y[e], scale, bias) : nothing;
                            to += a.ldc;
                        }
                    }
                }
                __syncwarp();
            }
            ug_fence_before();
            __syncwarp();
            if (lane == 0) {
                asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(q8p_at_leader(&drained[b]))
                             : "memory");
            }
        }
    }
    // copies and MMAs in flight end, in both blocks, before shared memory and tensor memory are released
    ug_fence_before();
    __syncthreads();
    cg::this_cluster().sync();
    if (rank == 0 && threadIdx.x == 0 && issued[1] < issued[0])
        for (int s = issued[1]; s < issued[0]; s++)
            if (!q8p_wait(&full[s % Q8P_STAGES], (uint32_t)((s / Q8P_STAGES) & 1))) break;
    __syncthreads();
    cg::this_cluster().sync();
    if (warp == 1) {
        ug_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <typename T> static cudaError_t q8pair_t(const Q8MatArgs& a, const CUtensorMap& levels, int device, int sms, cudaStream_t st) {
    static std::atomic<bool> ready[Q8_DEVICES];
    const auto kernel = dz_q8pair_kernel<T>;
    if (!ready[device].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Q8P_SMEM);
        if (e != cudaSuccess) return e;
        ready[device].store(true, std::memory_order_release);
    }
    CUtensorMap rows;
    const uint64_t dims[2] = {(uint64_t)a.K, (uint64_t)a.M}, strides[1] = {(uint64_t)a.lda};
    const uint32_t box[2] = {128, 128};
    if (!dz_encode_u8_map(&rows, a.a, 2, dims, strides, box)) return cudaErrorInvalidValue;
    const int ntiles = (a.N + Q8P_TILE - 1) / Q8P_TILE, mtiles = (a.M + Q8P_TILE - 1) / Q8P_TILE;
    const long long tiles = (long long)ntiles * mtiles;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * (tiles < sms / 2 ? tiles : sms / 2)));
    cfg.blockDim = dim3(Q8P_THREADS);
    cfg.dynamicSmemBytes = Q8P_SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, levels, rows, a, ntiles, mtiles);
}

template <typename T>
static cudaError_t q8gemm_n(const Q8MatArgs& a, const CUtensorMap& levels, const Q8Plan& plan, int device, int sms, cudaStream_t st) {
    if (plan.rows == 32) return q8gemm_t<T, 32>(a, levels, plan.parts, device, sms, st);
    if (plan.rows == 64) return q8gemm_t<T, 64>(a, levels, plan.parts, device, sms, st);
    if (plan.rows == 128) return q8gemm_t<T, 128>(a, levels, plan.parts, device, sms, st);
    return q8pair_t<T>(a, levels, device, sms, st);
}

cudaError_t dz_q8gemm_launch(const Q8MatArgs& a, const CUtensorMap& levels, const Q8Plan& plan, int type, int device, int sms,
                             cudaStream_t st) {
    if (type == DZ_TYPE_F32) return q8gemm_n<float>(a, levels, plan, device, sms, st);
    if (type == DZ_TYPE_F16) return q8gemm_n<__half>(a, levels, plan, device, sms, st);
    return q8gemm_n<__nv_bfloat16>(a, levels, plan, device, sms, st);
}

}  // namespace dz
