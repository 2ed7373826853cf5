// What the attention kernels over the 8-bit paged caches share (kv8attn.cu of
// few queries, kv8many.cu of many).
#pragma once
#include <atomic>

#include "async.cuh"
#include "kv8.cuh"
#include "qlevels.cuh"
#include "shim.cuh"

namespace dz {

constexpr int KV8_TILE = 32;       // tokens of a copy, all in one page
constexpr int KV8_CLUSTER = 16;    // blocks of a cluster at most
constexpr int KV8_DEVICES = 64;    // devices whose launch state is kept

// A box of 32 tokens' codes of a page's head.
__device__ __forceinline__ void kv8_copy(void* dst, const CUtensorMap* tm, int row, int page, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            dz_smem_addr(dst)),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(0), "r"(row), "r"(page), "r"(dz_smem_addr(bar))
        : "memory");
}

// The codes in bytes 0 and 2 (1 and 3) of x as two fp16.
template <bool ODD> __device__ __forceinline__ uint32_t kv8_widen(uint32_t x) {
    uint32_t biased;             // (x & bytes) ^ base, 1024 + 128 + code; one instruction, both constants in registers
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(biased) : "r"(ODD ? x >> 8 : x), "r"(0x00ff00ffu), "r"(0x64806480u));
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&biased), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&y);
}

__device__ __forceinline__ uint32_t kv8_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float kv8_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A weight is 2^15 times 2 to the power of its score x f less the largest one m.
// fma(x, f, 15 - m) does not round x f as m was, and rounds 15 - m: the largest
// weight is then off by as much as m's steps, half of one from 2^16 on 2^-8 and
// from 2^24 on 1, where it leaves fp16. From KV8_FAR on scores are rounded first,
// so that the largest weight is 2^15 exactly.
constexpr float KV8_FAR = 65536.0f;
__device__ __forceinline__ float kv8_far_power(float x, float f, float m) {
    return __fadd_rn(__fadd_rn(__fmul_rn(x, f), m == -INFINITY ? 0.0f : -m), 15.0f);
}

// What takes the weights' 2^15 off the sums, in the values' scales, so that sums
// stay in fp32's range as far as those of weights up to 1 do.
constexpr float KV8_LOWER = 0x1p-15f;

// Clusters of 1..16 blocks of a kernel that a device holds at once (a cluster
// stays within one GPC, so that larger ones leave SMs idle; 0: it cannot hold
// one). Asked once per kernel and device.
struct Kv8Room {
    std::atomic<bool> known{false};
    std::atomic<int> clusters[KV8_CLUSTER + 1];
};

// Code buffers as [pages][kv_heads page][head_dim] for kv8_copy: keys, values.
inline bool kv8_maps(const Kv8Cache& c, int head_dim, CUtensorMap (&maps)[2]) {
    const uint64_t rows = (uint64_t)c.kv_heads * c.page, width = (uint64_t)head_dim;
    const uint64_t dims[3] = {width, rows, (uint64_t)c.pages}, strides[2] = {width, rows * width};
    const uint32_t box[3] = {(uint32_t)head_dim, KV8_TILE, 1};
    return dz_encode_u8_map(&maps[0], c.k_codes, 3, dims, strides, box) && dz_encode_u8_map(&maps[1], c.v_codes, 3, dims, strides, box);
}

// kv8many.cu; `device` is below KV8_DEVICES.
[[nodiscard]] cudaError_t dz_kv8_many_launch(const Kv8AttnArgs& a, long long longest, int type, int head_dim, int device,
                                             cudaStream_t st);

}  // namespace dz
