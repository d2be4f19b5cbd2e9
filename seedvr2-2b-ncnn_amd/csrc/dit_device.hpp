// dit_device.hpp — device helpers of the GEMM kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace awa {

// A buffer resource over `bytes` from p with wave-uniform fields
// (readfirstlane returns int: each half of the address is taken back to
// uint32_t before widening, or a low word with bit 31 set would sign-extend
// into the high word; a resource the compiler cannot prove uniform makes it
// loop over the lanes at every access).  Loads past `bytes` read zeros and
// stores past it are dropped.
__device__ inline __amdgpu_buffer_rsrc_t uniform_rsrc(const void* p, uint32_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), 0,
                                             __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}

// Waits until at most N vector memory operations are outstanding.
template <int N>
__device__ inline void wait_vmem() {
    asm volatile("s_waitcnt vmcnt(%c0)" ::"n"(N) : "memory");
}

// The same, and no LDS operation.
template <int N>
__device__ inline void wait_vmem_lds() {
    asm volatile("s_waitcnt vmcnt(%c0) lgkmcnt(0)" ::"n"(N) : "memory");
}

}  // namespace awa
