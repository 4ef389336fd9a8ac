// Asynchronous copies of 4, 8 or 16 bytes from global to shared memory.  In the operators around the mixer every thread reads back
// what it asked for itself, so waiting for its own copies is all the ordering there is.
#pragma once
#include "mlstm_common.cuh"

namespace mlstm {

__device__ __forceinline__ unsigned shared_address(const void* p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }
// (16 bytes past the L1 cache, which the smaller ones have to go through)
template <int BYTES>
__device__ __forceinline__ void copy_async(unsigned shared, const void* global) {
    static_assert(BYTES == 4 || BYTES == 8 || BYTES == 16, "the sizes there are");
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared), "l"(global) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(shared), "l"(global), "n"(BYTES) : "memory");
}
// zeros where `there` is false (global is an address that may be read all the same)
template <int BYTES>
__device__ __forceinline__ void copy_async_or_zeros(unsigned shared, const void* global, bool there) {
    static_assert(BYTES == 4 || BYTES == 8, "as used");
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(shared), "l"(global), "n"(BYTES), "r"(there ? BYTES : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

}  // namespace mlstm
