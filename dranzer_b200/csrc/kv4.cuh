// The 4-bit ring caches (dz_kv4_t): what the append and attention kernels
// share.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace dz {

constexpr int KV4_GROUP = 64;   // elements of a row that share a scale
// Slots of a ring at most: attention counts them in 32 bits, up to two tiles past the end.
constexpr long long KV4_CAPACITY = INT32_MAX - 63;

struct Kv4Cache {
    uint8_t *k_codes, *v_codes;
    float *k_scales, *v_scales;
    int batch, kv_heads;
    long long capacity, sinks;
};

// The slot of position p >= 0.
__device__ __forceinline__ long long kv4_slot(long long p, long long sinks, long long ring) {
    if (p < sinks) return p;
    const long long r = p - sinks;
    if (((r | ring) >> 32) == 0) return sinks + (long long)((uint32_t)r % (uint32_t)ring);
    return sinks + r % ring;
}

// Whether a sequence is left out: its position is negative, or one whose slot
// arithmetic could leave 64 bits.
__device__ __forceinline__ bool kv4_skips(long long position) { return position < 0 || position >> 62; }

struct Kv4AppendArgs {
    Kv4Cache c;
    const long long* positions;
    long long pos_add;          // added to them (the model's caches count the step's token already)
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

struct Kv4AttnArgs {
    Kv4Cache c;
    const long long* positions;
    long long pos_add;          // added to them
    const void* q;
    void* out;
    long long ldq, ldo;
    int n_tokens, q_heads;
    float scale;
    long long window;
};

// base^(-2p / head_dim) for p < head_dim / 2, the rest 0 (all 0 for base 0).
void dz_kv4_frequencies(double base, size_t head_dim, double* freq);

[[nodiscard]] cudaError_t dz_kv4_append_launch(const Kv4AppendArgs& a, int type, int head_dim, int device, cudaStream_t st);
// Picks the kernel: kv4attn.cu for few pairs to a key head, kv4chunk.cu for many.
[[nodiscard]] cudaError_t dz_kv4_chunk_launch(const Kv4AttnArgs& a, int type, int head_dim, int device, cudaStream_t st);
[[nodiscard]] cudaError_t dz_kv4_attn_launch(const Kv4AttnArgs& a, int type, int head_dim, int device, cudaStream_t st);

}  // namespace dz
