// Helpers of the kernels on the 5th-generation tensor cores (tcgen05): bounded waits, issue by one lane, commits and fences.
#pragma once
#include "hp_common.cuh"

namespace hp {

// Bounded wait that lets the hardware park the warp: up to 2^20 attempts of up to a microsecond
__device__ __forceinline__ bool tc_wait(uint32_t bar, uint32_t parity, int* err) {
    for (uint32_t it = 0; it < (1u << 20); ++it) {
        uint32_t ok;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity), "r"(1000u) : "memory");
        if (ok) return true;
    }
    if (err) atomicExch(err, HP_ETIMEOUT);
    return false;
}
// one lane of a converged warp; unlike lane == 0 the compiler knows that a single thread issues what follows
__device__ __forceinline__ bool tc_elect() {
    uint32_t p;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

}  // namespace hp
