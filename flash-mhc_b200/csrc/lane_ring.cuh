// Two helpers of the streaming kernels: packed f32 pairs, and a shared-memory
// ring in which every lane prefetches the bytes that it will read itself.
//
// The ring replaces prefetching into registers: copies (cp.async) of the next
// iterations are in flight while the current one is computed, and the kernel's
// registers hold accumulators only.  A lane waits for its own copies and reads
// its own slots, so no barrier is involved; it refills a slot only after it has
// used what it read from it.  A slot that other lanes read as well (the row slots of
// the layer norm's backward) needs a warp barrier before its refill and after the wait.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <utility>

namespace fmhc {

// f(std::integral_constant<int, i>) for i = 0 .. N - 1: unrolled, with the index
// a constant (offsets of the asm below).
template <class F, int... I>
__device__ __forceinline__ void unrolled_(F &&f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void unrolled(F &&f) {
  unrolled_(f, std::make_integer_sequence<int, N>{});
}

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
// The same with a shared-memory address plus a constant.
template <int BYTES, int OFF>
__device__ __forceinline__ void copy_async_at(uint32_t dst, const void *src) {
  static_assert(BYTES == 16 || BYTES == 8, "copy size");
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0 + %2], [%1], 16;" ::"r"(dst), "l"(src), "n"(OFF) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0 + %2], [%1], 8;" ::"r"(dst), "l"(src), "n"(OFF) : "memory");
}
// Four bytes, or the first `valid` of them and zeros.
__device__ __forceinline__ void copy_async4(uint32_t dst, const void *src, int valid = 4) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
}
// Shared-memory loads at an address plus a constant.
template <int OFF>
__device__ __forceinline__ uint4 load_shared16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a), "n"(OFF)
               : "memory");
  return v;
}
template <int OFF>
__device__ __forceinline__ uint2 load_shared8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2 + %3];" : "=r"(v.x), "=r"(v.y) : "r"(a), "n"(OFF) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t load_shared_u8(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float load_shared_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float2 load_shared_f32x2(uint32_t a) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Wait until at most N of this thread's latest groups are still in flight.
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace fmhc
