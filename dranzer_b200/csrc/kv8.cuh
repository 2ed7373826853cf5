// The 8-bit paged caches (dz_kv8_t): what the append and attention kernels
// share.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace dz {

// Positions that a table reaches at most: attention counts them in 32 bits, tiles
// of 32 tokens with a sign, those of 128, which may pass the end, without.
constexpr long long KV8_REACH = INT32_MAX - 63;

struct Kv8Cache {
    int8_t *k_codes, *v_codes;
    float *k_scales, *v_scales;
    const int32_t* table;
    int batch, kv_heads, pages, page, table_pages;
};

// Whether a sequence is left out: its position is negative, or one whose
// arithmetic could leave 64 bits.
__device__ __forceinline__ bool kv8_skips(long long position) { return position < 0 || position >> 62; }

struct Kv8AppendArgs {
    Kv8Cache c;
    const long long* positions;
    const void *q, *k, *v;
    void *q_out, *k_out, *v_out;
    long long ldq, ldk, ldv, ldqo, ldko, ldvo;
    const float *q_gain, *k_gain;
    double eps;
    int n_tokens, q_heads;
    int rope;                   // rotate at all
    int halves;                 // DZ_ROPE_HALVES
    double freq[64];            // base^(-2p / head_dim), p < head_dim / 2
};

struct Kv8AttnArgs {
    Kv8Cache c;
    const long long* positions;
    const void* q;
    void* out;
    long long ldq, ldo;
    int n_tokens, q_heads;
    float scale;
    long long window;
};

[[nodiscard]] cudaError_t dz_kv8_append_launch(const Kv8AppendArgs& a, int type, int head_dim, int device, cudaStream_t st);
// `longest`: the most tokens that a sequence is thought to hold.
[[nodiscard]] cudaError_t dz_kv8_attn_launch(const Kv8AttnArgs& a, long long longest, int type, int head_dim, int device,
                                             cudaStream_t st);

}  // namespace dz
