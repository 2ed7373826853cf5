// Shared-memory addresses and mbarriers, for kernels that wait for asynchronous
// copies.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace dz {

__device__ __forceinline__ uint32_t dz_smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ uint64_t dz_global_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// mbarrier helpers (count-1 barriers completed by expect_tx + bulk copies)
__device__ __forceinline__ void dz_mbar_init(uint64_t* bar) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(dz_smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void dz_mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(dz_smem_addr(bar)), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ bool dz_mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(dz_smem_addr(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
// Bounded wait (about one second). False when it gave up. The timer is read
// only once the phase has not completed on the first tries (a global-timer
// read costs far more than a try_wait that succeeds).
__device__ __forceinline__ bool dz_mbar_wait(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
    for (int i = 0; i < 4; i++)
        if (dz_mbar_test(bar, parity)) return true;
    const uint64_t t0 = dz_global_ns();
    for (unsigned i = 0;; i++) {
        if (dz_mbar_test(bar, parity)) return true;
        if ((i & 255u) == 255u && dz_global_ns() - t0 > 1000000000ull) return false;
    }
}

}  // namespace dz
