// Two helpers of the streaming kernels: packed f32 pairs, and a shared-memory
// ring in which every lane prefetches the bytes that it will read itself.
//
// The ring replaces prefetching into registers: copies (cp.async) of the next
// iterations are in flight while the current one is computed, and the kernel's
// registers hold accumulators only.  A lane waits for its own copies and reads
// its own slots, so no barrier is involved; it refills a slot only after it has
// used what it read from it.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace fmhc {

// ------------------------------------------------- two f32 in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long &>(d))
      : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)),
        "l"(reinterpret_cast<unsigned long long &>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long &>(d))
      : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long &>(d))
      : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// ------------------------------------------------------------------- copies
__device__ __forceinline__ uint32_t shared_addr(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
// Global -> shared, asynchronous; BYTES 16 or 8, both addresses aligned to it.
template <int BYTES>
__device__ __forceinline__ void copy_async(void *dst, const void *src) {
  static_assert(BYTES == 16 || BYTES == 8, "copy size");
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared_addr(dst)), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(shared_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Wait until at most N of this thread's latest groups are still in flight.
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace fmhc
