// Loads that put their data into LDS by themselves.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nnb {

// A pointer that all lanes agree on, in scalar registers.
template <typename T> __device__ __forceinline__ T *uniform(T *p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return reinterpret_cast<T *>((uint64_t)hi << 32 | lo);
}

// 16 bytes a lane from base + offset to 1 KB of LDS at `to` (base and `to` uniform).  In assembly because the compiler,
// which cannot tell the parts of a ring of buffers apart, would wait for every load in flight before every read of LDS;
// the kernels' own waits in front of their barriers (wait_and_meet) are the only ones needed.
// The clobber keeps it from standing between a use of m0 and what set it; that the register is reserved, which the
// compiler warns of, only means that no value lives there for long.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(const void *base, uint32_t offset, void *to) {
    const uint32_t m0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)to;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :: "v"(offset), "s"(base), "s"(__builtin_amdgcn_readfirstlane(m0)) : "memory", "m0");
}
#pragma clang diagnostic pop

// All but the wave's last IN_FLIGHT memory operations and all its LDS reads are done; after the barrier everybody's are.
template <int IN_FLIGHT> __device__ __forceinline__ void wait_and_meet() {
    static_assert(IN_FLIGHT < 64, "the counter's range");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(IN_FLIGHT) : "memory");
}

}  // namespace nnb
