// Rows in 8 bits: one f32 scale per row and one int8 code per value, the form in
// which the 8-bit linear layer takes activations and weights.
//
// With a = max |v| over the row, at least kLeast:
//   scale = a / 127,  code = RNE(v * (127 / a)),  value = code * scale
// A row that holds an infinity or a NaN has codes 0 and the scale NaN: what is
// computed from it is NaN in every place.  kLeast keeps 127 / a finite; a row of
// zeros has codes 0 and the scale kLeast / 127.
//
// Unlike the 8-bit checkpoints (act8.cuh: blocks of 32, power-of-two scales, no
// rounding but the codes') the scale is as fine as the row allows and constant
// along it, so that it leaves the sum of products of a linear layer.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace fmhc {
namespace rows8 {

constexpr float kLeast = 7.888609052210118e-31f;  // 2^-100

// The row's scale and the factor of its codes, from the f32 bits of its largest
// magnitude (an infinity or a NaN has the largest bits).
struct RowScale {
  float scale, inv;
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax) {
  if (amax >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.f};
  const float a = fmaxf(__uint_as_float(amax), kLeast);
  return {__fdiv_rn(a, 127.f), __fdiv_rn(127.f, a)};
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// 1.5 * 2^23 + q rounds |q| <= 127 to the nearest even integer, whose two's
// complement is the low byte.  A row with inv = 0 has codes 0, whatever v is.
__device__ __forceinline__ uint32_t code_bits(float v, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.f));
}
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d, float inv) {
  const uint32_t lo = __byte_perm(code_bits(a, inv), code_bits(b, inv), 0x0040);
  const uint32_t hi = __byte_perm(code_bits(c, inv), code_bits(d, inv), 0x0040);
  return inv == 0.f ? 0u : __byte_perm(lo, hi, 0x5410);
}
__device__ __forceinline__ int8_t code1(float v, float inv) {
  return inv == 0.f ? int8_t(0) : int8_t(code_bits(v, inv) & 0xffu);
}
// Eight codes to an 8-byte aligned place.
__device__ __forceinline__ void store_codes8(int8_t *p, const float (&f)[8], float inv) {
  __stcs(reinterpret_cast<uint2 *>(p), make_uint2(code4(f[0], f[1], f[2], f[3], inv), code4(f[4], f[5], f[6], f[7], inv)));
}

}  // namespace rows8
}  // namespace fmhc
