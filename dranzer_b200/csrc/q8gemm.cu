// Products of 8-bit rows with a quantized matrix on the tensor cores
// (q8matmul.cuh): D[n][m] = sum_k level[n][k] a[m][k] in kind::i8 MMAs, the
// matrix's columns as the 128 lanes of tensor memory and the rows as its
// columns, so that an output row is written by the lanes of a warp side by
// side. Both operands are K-major and come by TMA with the 128-byte swizzle,
// what lies past the rows or past k as zeros.
#define DZ_KERNEL_LINKAGE static   // the helper headers' own kernels stay private to dz_cuda.cu
#include "umma.cuh"

#include <atomic>
#include <cooperative_groups.h>

#include "q8matmul.cuh"
#include "qlevels.cuh"

namespace dz {

namespace cg = cooperative_groups;

constexpr int Q8G_THREADS = 256;
constexpr uint32_t Q8G_A_BYTES = 128 * 128;      // levels of a stage

template <int TN> struct Q8gShape {
    static constexpr uint32_t B_BYTES = TN * 128;
    static constexpr uint32_t STAGE = Q8G_A_BYTES + B_BYTES;
    // two blocks to an SM for narrow tiles, one for wide ones
    static constexpr int STAGES = TN <= 64 ? (int)(100 * 1024 / STAGE) : (int)(200 * 1024 / STAGE);
    static constexpr size_t SMEM = (size_t)STAGES * STAGE + 1024 + 256;
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
__global__ void __launch_bounds__(Q8G_THREADS, TN <= 64 ? 2 : 1)
    dz_q8gemm_kernel(const __grid_constant__ CUtensorMap tm_levels, const __grid_constant__ CUtensorMap tm_rows,
                     const __grid_constant__ Q8MatArgs a, int parts) {
    using S = Q8gShape<TN>;
    extern __shared__ __align__(1024) uint8_t q8g_raw[];
    uint8_t* sm = q8g_raw + ((1024u - (dz_smem_addr(q8g_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + (size_t)S::STAGES * S::STAGE);
    uint64_t* empty = full + S::STAGES;
    uint64_t* accum = empty + S::STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accum + 1);
    int* progress = reinterpret_cast<int*>(tmem_slot + 1);       // stages issued, consumed; failed
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = (int)(blockIdx.x % (unsigned)parts), tile = (int)(blockIdx.x / (unsigned)parts);
    const int n0 = tile * 128, m0 = blockIdx.y * TN;
    const int kb0 = (int)((long long)a.nkb * part / parts), nkb = (int)((long long)a.nkb * (part + 1) / parts) - kb0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; s++) {
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
        if (lane == 0) {
            // the levels of the first stages are no kernel's output and go out before the one before has ended
            const int pre = nkb < S::STAGES ? nkb : S::STAGES;
            for (int kb = 0; kb < pre; kb++) {
                dz_mbar_expect_tx(&full[kb], S::STAGE);
                ug_tma_4d(sm + (size_t)kb * S::STAGE, &tm_levels, 0, 0, kb0 + kb, tile, &full[kb]);
            }
            asm volatile("griddepcontrol.wait;" ::: "memory");
            int kb = 0;
            for (; kb < nkb; kb++) {
                const int s = kb % S::STAGES;
                if (kb >= S::STAGES && !dz_mbar_wait(&empty[s], (uint32_t)(((kb / S::STAGES) - 1) & 1))) {
                    progress[2] = 1;
                    break;
                }
                uint8_t* to = sm + (size_t)s * S::STAGE;
                if (kb >= pre) {
                    dz_mbar_expect_tx(&full[s], S::STAGE);
                    ug_tma_4d(to, &tm_levels, 0, 0, kb0 + kb, tile, &full[s]);
                }
                q8g_tma_2d(to + Q8G_A_BYTES, &tm_rows, (kb0 + kb) * 128, m0, &full[s]);
            }
            progress[0] = kb;
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            int kb = 0;
            for (; kb < nkb; kb++) {
                const int s = kb % S::STAGES;
                if (!dz_mbar_wait(&full[s], (uint32_t)((kb / S::STAGES) & 1))) {
                    progress[2] = 1;
                    break;
                }
                ug_fence_after();
                const uint32_t at = dz_smem_addr(sm + (size_t)s * S::STAGE);
#pragma unroll
                for (int kk = 0; kk < 4; kk++)
                    ug_mma(tmem, ug_desc_kmajor(at + kk * 32), ug_desc_kmajor(at + Q8G_A_BYTES + kk * 32), q8g_idesc<TN>(),
                           (kb > 0 || kk > 0) ? 1u : 0u);
                ug_commit(&empty[s]);
            }
            progress[1] = kb;
            ug_commit(accum);
        }
        __syncwarp();
    }
    const bool ok = dz_mbar_wait(accum, 0);
    ug_fence_after();
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the rows' scales
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
        const int n = n0 + (threadIdx.x & 127);
        if (n < a.N) {
            const float scale = a.col_scale[n], bias = a.bias ? a.bias[n] : 0.0f;
            for (int r = first + (threadIdx.x >> 7); r < last; r += 2) {
                int sum = 0;
                for (int p = 0; p < parts; p++) sum += cluster.map_shared_rank(sums, p)[r * 128 + (threadIdx.x & 127)];
                c[(m0 + r) * a.ldc + n] = lost ? nothing : q8_finish<T>(sum, a.a_scales[m0 + r], scale, bias);
            }
        }
        cluster.sync();                      // no block ends while another reads its shared memory
    }
    // copies and MMAs in flight end before the shared memory and the tensor memory are released
    ug_fence_before();
    if (threadIdx.x == 0 && progress[2]) {
        for (int kb = progress[1]; kb < progress[0]; kb++)
            if (!dz_mbar_wait(&full[kb % S::STAGES], (uint32_t)((kb / S::STAGES) & 1))) break;
        dz_mbar_wait(accum, 0);
    }
    __syncthreads();
    if (warp == 1) {
        ug_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)TN) : "memory");
    }
}

template <typename T, int TN>
static cudaError_t q8gemm_t(const Q8MatArgs& a, const CUtensorMap& levels, int device, int sms, cudaStream_t st) {
    static std::atomic<bool> ready[Q8_DEVICES];
    using S = Q8gShape<TN>;
    const auto kernel = dz_q8gemm_kernel<T, TN>;
    if (!ready[device].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM);
        if (e != cudaSuccess) return e;
        ready[device].store(true, std::memory_order_release);
    }
    CUtensorMap rows;
    const uint64_t dims[2] = {(uint64_t)a.K, (uint64_t)a.M}, strides[1] = {(uint64_t)a.lda};
    const uint32_t box[2] = {128, (uint32_t)TN};
    if (!dz_encode_u8_map(&rows, a.a, 2, dims, strides, box)) return cudaErrorInvalidValue;
    const int tiles = (a.N + 127) / 128, mtiles = (a.M + TN - 1) / TN;
    int parts = 1;
    const int slots = sms * (TN <= 64 ? 2 : 1);
    while (parts < 8 && 2 * parts * tiles * mtiles <= slots && a.nkb >= 4 * parts) parts *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * parts), (unsigned)mtiles);
    cfg.blockDim = dim3(Q8G_THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, levels, rows, a, parts);
}

template <typename T> static cudaError_t q8gemm_n(const Q8MatArgs& a, const CUtensorMap& levels, int device, int sms, cudaStream_t st) {
    if (a.M <= 32) return q8gemm_t<T, 32>(a, levels, device, sms, st);
    if (a.M <= 64) return q8gemm_t<T, 64>(a, levels, device, sms, st);
    if (a.M <= 128) return q8gemm_t<T, 128>(a, levels, device, sms, st);
    return q8gemm_t<T, 256>(a, levels, device, sms, st);
}

cudaError_t dz_q8gemm_launch(const Q8MatArgs& a, const CUtensorMap& levels, int type, int device, int sms, cudaStream_t st) {
    if (type == DZ_TYPE_F32) return q8gemm_n<float>(a, levels, device, sms, st);
    if (type == DZ_TYPE_F16) return q8gemm_n<__half>(a, levels, device, sms, st);
    return q8gemm_n<__nv_bfloat16>(a, levels, device, sms, st);
}

}  // namespace dz
