// 8-bit activation checkpoints: the format and its device helpers.
//
// A row of C values is cut into blocks of 32 (the last may be shorter).  Each
// block has one scale byte e, standing for 2^(e - 127), and one 8-bit code per
// value.  With a = max |x| over the block and M the largest code (127 for
// int8, 448 for e4m3):
//   e    = the smallest byte with a <= M 2^(e - 127), at most 254 - floor(log2 M)
//          (so M 2^(e - 127) is a finite f32; larger values saturate)
//   code = RNE(x / 2^(e - 127)), kept in [-M, M]
//   value = code 2^(e - 127)
// A block that holds an infinity or a NaN has e = 255 and codes 0 and stands
// for NaN in every place: a non-finite activation is never hidden.
//
// The scale is a power of two, so x / scale and code * scale are exact in f32
// and e comes from the bits of a alone: the same bytes on every path, no
// division, and an int8 or e4m3 value is exact in bf16 (at most 7 significant
// bits), which is what lets a checkpoint feed a bf16 tensor-core product.  The
// price against a scale of a / M is at most one bit of the code range.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "fmhc_common.cuh"
#include "lane_ring.cuh"

namespace fmhc {
namespace act8 {

constexpr int kBlock = 32;           // values per scale byte
constexpr int kInt8 = 0, kE4m3 = 1;  // FMHC_ACT8_INT8, FMHC_ACT8_E4M3
constexpr int kNone = -1;            // no 8-bit copy

// a <= M 2^k  <=>  the significand of a is at most M's, after which a's
// exponent carries: adding kCarry to the f32 bits of a does exactly that.
template <int FMT> struct Format;
template <> struct Format<kInt8> {
  static constexpr uint32_t kCarry = 0x1FFFFu;  // M = 1.984375 * 2^6
  static constexpr uint32_t kTop = 6;
  static constexpr float kMax = 127.f;
};
template <> struct Format<kE4m3> {
  static constexpr uint32_t kCarry = 0x1FFFFFu;  // M = 1.75 * 2^8
  static constexpr uint32_t kTop = 8;
  static constexpr float kMax = 448.f;
};

// Scale byte of a block whose largest magnitude has the f32 bits `amax`.
template <int FMT>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  const uint32_t e = min((amax + Format<FMT>::kCarry) >> 23, 254u);
  const uint32_t s = e > Format<FMT>::kTop ? e - Format<FMT>::kTop : 0u;
  return amax >= 0x7f800000u ? 255u : s;
}

// 2^(e - 127); 2^-127 is subnormal, 255 gives NaN.
__device__ __forceinline__ float scale_value(uint32_t e) {
  uint32_t b = e << 23;
  if (e == 0u) b = 0x00400000u;
  if (e == 255u) b = 0x7fc00000u;
  return __uint_as_float(b);
}

// The scale bytes below this one need no care in encode4: no value of their
// block is above M times the scale, and none is infinite or NaN.
template <int FMT> constexpr uint32_t kTopScale = 254u - Format<FMT>::kTop;

// Four values -> four codes in one word (value 0 in the lowest byte).  CARE: the
// scale byte may be kTopScale (saturate) or 255 (codes 0).
template <int FMT, bool CARE>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, uint32_t e) {
  const float inv = __uint_as_float((254u - (CARE ? min(e, kTopScale<FMT>) : e)) << 23);
  float v[4] = {a * inv, b * inv, c * inv, d * inv};
  uint32_t w;
  if constexpr (FMT == kInt8) {
    if constexpr (CARE) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = fminf(fmaxf(v[i], -Format<FMT>::kMax), Format<FMT>::kMax);
    }
    // 1.5 * 2^23 + q rounds q to the nearest even integer; its low byte is
    // that integer in two's complement.
    uint32_t m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = __float_as_uint(v[i] + 12582912.f);
    w = __byte_perm(__byte_perm(m[0], m[1], 0x0040), __byte_perm(m[2], m[3], 0x0040), 0x5410);
  } else {
    uint16_t lo, hi;  // round to nearest even, saturating at +-448
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(v[1]), "f"(v[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(v[3]), "f"(v[2]));
    w = uint32_t(lo) | (uint32_t(hi) << 16);
  }
  return CARE && e == 255u ? 0u : w;
}

// One word of codes -> four unscaled f32 values (exact).
template <int FMT>
__device__ __forceinline__ void decode4(uint32_t w, float (&f)[4]) {
  if constexpr (FMT == kInt8) {
    const uint32_t u = w ^ 0x80808080u;  // code + 128 in 0..255
#pragma unroll
    for (int i = 0; i < 4; ++i)           // 2^23 + (code + 128), then minus the offset
      f[i] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650u + i)) - 8388736.f;
  } else {
    uint32_t a, b;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(a) : "h"(uint16_t(w)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(b) : "h"(uint16_t(w >> 16)));
    const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&a));
    const float2 q = __half22float2(*reinterpret_cast<const __half2 *>(&b));
    f[0] = p.x; f[1] = p.y; f[2] = q.x; f[3] = q.y;
  }
}
// The same as two pairs.
template <int FMT>
__device__ __forceinline__ void decode4x2(uint32_t w, float2 &a, float2 &b) {
  if constexpr (FMT == kInt8) {
    const uint32_t u = w ^ 0x80808080u, m = 0x4b000000u;
    const float2 o = both(-8388736.f);
    a = add2(make_float2(__uint_as_float(__byte_perm(u, m, 0x7650)), __uint_as_float(__byte_perm(u, m, 0x7651))), o);
    b = add2(make_float2(__uint_as_float(__byte_perm(u, m, 0x7652)), __uint_as_float(__byte_perm(u, m, 0x7653))), o);
  } else {
    float f[4];
    decode4<FMT>(w, f);
    a = make_float2(f[0], f[1]);
    b = make_float2(f[2], f[3]);
  }
}
template <int FMT>
__device__ __forceinline__ float decode1(uint8_t c) {
  if constexpr (FMT == kInt8) {
    return __uint_as_float(0x4b000000u | (c ^ 0x80u)) - 8388736.f;  // as in decode4
  } else {
    float f[4];
    decode4<FMT>(uint32_t(c), f);
    return f[0];
  }
}

// Scale byte -> the factor that widen4 takes: 2^(e - 127) as two bf16 or as f32.
template <int FMT>
__device__ __forceinline__ uint32_t widen_factor(uint32_t e) {
  const uint32_t f = __float_as_uint(scale_value(e));
  return FMT == kInt8 ? __byte_perm(f, 0, 0x3232) : f;
}

// Four codes -> four bf16 values (exact: at most 7 significant bits).
template <int FMT>
__device__ __forceinline__ uint2 widen4(uint32_t w, uint32_t factor) {
  if constexpr (FMT == kInt8) {
    // 0x4300 | code is, as bf16, 128 + (code & 127) once bit 7 is cleared, and
    // 128 or 256 (for a negative code) once bits 0-6 are: the difference is the
    // code.  Two codes per instruction, exact in bf16.
    uint32_t o[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t p = __byte_perm(w, 0x43434343u, i ? 0x7372 : 0x7170);
      const uint32_t hi = p & 0xff7fff7fu, lo = p & 0xff80ff80u;
      const __nv_bfloat162 v = __hmul2(__hsub2(reinterpret_cast<const __nv_bfloat162 &>(hi),
                                               reinterpret_cast<const __nv_bfloat162 &>(lo)),
                                       reinterpret_cast<const __nv_bfloat162 &>(factor));
      o[i] = reinterpret_cast<const uint32_t &>(v);
    }
    return make_uint2(o[0], o[1]);
  } else {
    float f[4];
    decode4<FMT>(w, f);
    const float2 s = both(__uint_as_float(factor));
    const float2 a = mul2(make_float2(f[0], f[1]), s), b = mul2(make_float2(f[2], f[3]), s);
    return make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(b.x, b.y));
  }
}

// Eight codes loaded as one access, and widened to scaled f32 values.
__device__ __forceinline__ uint2 ld_codes8(const uint8_t *p) {
  return __ldcs(reinterpret_cast<const uint2 *>(p));
}
template <int FMT>
__device__ __forceinline__ void restore(uint2 c, float s, float (&f)[8]) {
  float a[4], b[4];
  decode4<FMT>(c.x, a);
  decode4<FMT>(c.y, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = a[i] * s;
    f[i + 4] = b[i] * s;
  }
}

// ---------------------------------------------------------------------------
// Elements of the three activation types: eight consecutive ones as raw words,
// their f32 values, and one at a time.
// ---------------------------------------------------------------------------
template <class E> struct Elem;
template <> struct Elem<__nv_bfloat16> {
  using Raw = uint4;
  static __device__ __forceinline__ void widen(const Raw &r, float (&f)[8]) {
    f[0] = bf16lo(r.x); f[1] = bf16hi(r.x); f[2] = bf16lo(r.y); f[3] = bf16hi(r.y);
    f[4] = bf16lo(r.z); f[5] = bf16hi(r.z); f[6] = bf16lo(r.w); f[7] = bf16hi(r.w);
  }
  static __device__ __forceinline__ Raw narrow(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  }
  static __device__ __forceinline__ float widen1(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 narrow1(float f) { return __float2bfloat16_rn(f); }
  static __device__ __forceinline__ float fit(float f) { return f; }
};
template <> struct Elem<__half> {
  using Raw = uint4;
  static __device__ __forceinline__ void widen(const Raw &r, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ Raw narrow(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float widen1(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half narrow1(float f) { return __float2half_rn(f); }
  // A restored value may lie just above the largest f16 (65504 is restored
  // from the code 64 as 65536): keep it finite.  NaN passes.
  static __device__ __forceinline__ float fit(float f) {
    f = f > 65504.f ? 65504.f : f;
    return f < -65504.f ? -65504.f : f;
  }
};
template <> struct Elem<float> {
  struct Raw { uint4 a, b; };
  static __device__ __forceinline__ void widen(const Raw &r, float (&f)[8]) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
  }
  static __device__ __forceinline__ Raw narrow(const float (&f)[8]) {
    Raw r;
    r.a = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                     __float_as_uint(f[3]));
    r.b = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]),
                     __float_as_uint(f[7]));
    return r;
  }
  static __device__ __forceinline__ float widen1(float v) { return v; }
  static __device__ __forceinline__ float narrow1(float f) { return f; }
  static __device__ __forceinline__ float fit(float f) { return f; }
};

template <class E>
__device__ __forceinline__ typename Elem<E>::Raw ld8(const E *p) {
  if constexpr (sizeof(E) == 2) {
    return __ldcs(reinterpret_cast<const uint4 *>(p));
  } else {
    typename Elem<E>::Raw r;
    r.a = __ldcs(reinterpret_cast<const uint4 *>(p));
    r.b = __ldcs(reinterpret_cast<const uint4 *>(p) + 1);
    return r;
  }
}
template <class E>
__device__ __forceinline__ void st8(E *p, const float (&f)[8]) {
  if constexpr (sizeof(E) == 2) {
    __stcs(reinterpret_cast<uint4 *>(p), Elem<E>::narrow(f));
  } else {
    const typename Elem<E>::Raw r = Elem<E>::narrow(f);
    __stcs(reinterpret_cast<uint4 *>(p), r.a);
    __stcs(reinterpret_cast<uint4 *>(p) + 1, r.b);
  }
}

// Largest magnitude among eight raw values, as f32 bits.  Magnitudes of a
// floating type are ordered like their bits, infinity and NaN above the rest,
// so 16-bit values are compared two at a time without widening them.
template <class E>
__device__ __forceinline__ uint32_t amax8_raw(const typename Elem<E>::Raw &r) {
  if constexpr (sizeof(E) == 2) {
    const uint32_t k = 0x7fff7fffu;
    const uint32_t m = __vmaxu2(__vmaxu2(r.x & k, r.y & k), __vmaxu2(r.z & k, r.w & k));
    const uint32_t h = max(m & 0xffffu, m >> 16);
    if constexpr (std::is_same<E, __nv_bfloat16>::value) return h << 16;
    else return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(h))));
  } else {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m;
  }
}

// The same over the four lanes that share a block (lanes 4k .. 4k+3, eight
// values each); every lane of the warp takes part.
__device__ __forceinline__ uint32_t amax_block(uint32_t m) {
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
}

// Encodes eight values of a block with scale byte e, or one.
template <int FMT>
__device__ __forceinline__ uint2 encode8(const float (&f)[8], uint32_t e) {
  if (e < kTopScale<FMT>)
    return make_uint2(encode4<FMT, false>(f[0], f[1], f[2], f[3], e), encode4<FMT, false>(f[4], f[5], f[6], f[7], e));
  return make_uint2(encode4<FMT, true>(f[0], f[1], f[2], f[3], e), encode4<FMT, true>(f[4], f[5], f[6], f[7], e));
}
template <int FMT>
__device__ __forceinline__ uint8_t encode1(float f, uint32_t e) {
  if constexpr (FMT == kInt8) {  // encode4 of one value
    const float v = f * __uint_as_float((254u - min(e, kTopScale<FMT>)) << 23);
    const float c = fminf(fmaxf(v, -Format<FMT>::kMax), Format<FMT>::kMax);
    return e == 255u ? 0 : uint8_t(__float_as_uint(c + 12582912.f));
  } else {
    return uint8_t(encode4<FMT, true>(f, 0.f, 0.f, 0.f, e));
  }
}

}  // namespace act8
}  // namespace fmhc

// Run-time element type (fmhc_dtype) and code format -> template arguments E
// and FMT; the caller has checked both.
#define FMHC_DISPATCH_ELEM(DTYPE, ...)                          \
  do {                                                          \
    if ((DTYPE) == 0) { using E = float; __VA_ARGS__; }         \
    else if ((DTYPE) == 1) { using E = __nv_bfloat16; __VA_ARGS__; } \
    else { using E = __half; __VA_ARGS__; }                     \
  } while (0)
#define FMHC_DISPATCH_FMT(FMT_RT, ...)                                          \
  do {                                                                          \
    if ((FMT_RT) == ::fmhc::act8::kInt8) { constexpr int FMT = ::fmhc::act8::kInt8; __VA_ARGS__; } \
    else { constexpr int FMT = ::fmhc::act8::kE4m3; __VA_ARGS__; }              \
  } while (0)
