// The stream mixings K3 and K4 with 8-bit activation checkpoints (format:
// act8.cuh): the forwards that also write the codes of what they read, and the
// backwards that read codes where k3k4_stream.cu reads bf16.
//
// Work mapping as in k3k4_stream.cu: one warp per token, lanes walk C in chunks
// of eight values.  Four neighbouring lanes hold one block of 32 values, so a
// block's maximum takes two shuffles, and lane 4k writes or reads its scale.
#include "act8.cuh"
#include "fmhc_launch.h"
#include "grid.cuh"

namespace fmhc {

using namespace act8;
using bf16 = __nv_bfloat16;

namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------- K3 forward
//   out[t,c] = bf16( sum_j h_pre[t,j] x[t,j,c] ), and x in 8 bits.
template <int FMT>
__global__ void __launch_bounds__(kThreads)
k3_fwd_q8_kernel(const bf16 *__restrict__ x, const float4 *__restrict__ hp, bf16 *__restrict__ out,
                 uint8_t *__restrict__ codes, uint8_t *__restrict__ scales, int64_t T, int C) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  const int nchunk = C / 8, nb = (C + kBlock - 1) / kBlock;
  for (int64_t t = warp; t < T; t += nwarps) {
    const float4 h = __ldg(hp + t);
    const float hj[4] = {h.x, h.y, h.z, h.w};
    const bf16 *xr = x + t * 4 * C;
    for (int c0 = 0; c0 < nchunk; c0 += 32) {
      const int c = c0 + lane;
      const bool in = c < nchunk;
      uint4 a[4] = {};
      if (in) {
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = ld8(xr + j * C + c * 8);
      }
      float o[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[8];
        Elem<bf16>::widen(a[j], f);
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = j ? fmaf(hj[j], f[k], o[k]) : hj[0] * f[k];
        const uint32_t e = scale_byte<FMT>(amax_block(amax8(f)));
        const int64_t row = t * 4 + j;
        if (in) {
          __stcs(reinterpret_cast<uint2 *>(codes + row * C + c * 8), encode8<FMT>(f, e));
          if ((lane & 3) == 0) __stcs(scales + row * nb + (c >> 2), uint8_t(e));
        }
      }
      if (in) st8(out + t * C + c * 8, o);
    }
  }
}

// ---------------------------------------------------------------- K4 forward
//   out[t,i,c] = bf16( sum_j H[t,i,j] x[t,j,c] + h_post[t,i] lo[t,c] ), and lo
//   in 8 bits.
template <int FMT>
__global__ void __launch_bounds__(kThreads)
k4_fwd_q8_kernel(const bf16 *__restrict__ x, const bf16 *__restrict__ lo,
                 const float4 *__restrict__ H, const float4 *__restrict__ hpost,
                 bf16 *__restrict__ out, uint8_t *__restrict__ codes,
                 uint8_t *__restrict__ scales, int64_t T, int C) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  const int nchunk = C / 8, nb = (C + kBlock - 1) / kBlock;
  for (int64_t t = warp; t < T; t += nwarps) {
    float Hm[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 r = __ldg(H + t * 4 + i);
      Hm[i][0] = r.x; Hm[i][1] = r.y; Hm[i][2] = r.z; Hm[i][3] = r.w;
    }
    const float4 hp4 = __ldg(hpost + t);
    const float hp[4] = {hp4.x, hp4.y, hp4.z, hp4.w};
    const bf16 *xr = x + t * 4 * C;
    for (int c0 = 0; c0 < nchunk; c0 += 32) {
      const int c = c0 + lane;
      const bool in = c < nchunk;
      uint4 a[4] = {}, l = {};
      if (in) {
        l = ld8(lo + t * C + c * 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = ld8(xr + j * C + c * 8);
      }
      float fl[8], fx[4][8];
      Elem<bf16>::widen(l, fl);
#pragma unroll
      for (int j = 0; j < 4; ++j) Elem<bf16>::widen(a[j], fx[j]);
      const uint32_t e = scale_byte<FMT>(amax_block(amax8(fl)));
      if (in) {
        __stcs(reinterpret_cast<uint2 *>(codes + t * C + c * 8), encode8<FMT>(fl, e));
        if ((lane & 3) == 0) __stcs(scales + t * nb + (c >> 2), uint8_t(e));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float o[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {  // in the order of fmhc_k4_fwd
            float acc = hp[i] * fl[k];
            acc = fmaf(Hm[i][0], fx[0][k], acc);
            acc = fmaf(Hm[i][1], fx[1][k], acc);
            acc = fmaf(Hm[i][2], fx[2][k], acc);
            o[k] = fmaf(Hm[i][3], fx[3][k], acc);
          }
          st8(out + (t * 4 + i) * C + c * 8, o);
        }
      }
    }
  }
}

// VEC bf16 values -> f32 (VEC 8 or 1).
template <int VEC>
__device__ __forceinline__ void load_f32(const bf16 *p, float (&f)[VEC]) {
  if constexpr (VEC == 8) Elem<bf16>::widen(ld8(p), f);
  else f[0] = Elem<bf16>::widen1(*p);
}

// --------------------------------------------------------------- K3 backward
//   grad_h[t,j] = sum_c x8[t,j,c] go[t,c]
template <int FMT, int VEC>
__global__ void __launch_bounds__(kThreads)
k3_bwd_q8_kernel(const bf16 *__restrict__ go, const uint8_t *__restrict__ codes,
                 const uint8_t *__restrict__ scales, float *__restrict__ gh, int64_t T, int C) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  const int nchunk = C / VEC, nb = (C + kBlock - 1) / kBlock;
  for (int64_t t = warp; t < T; t += nwarps) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c = lane; c < nchunk; c += 32) {
      Codes<VEC> q[4];
      uint32_t e[4];
      float g[VEC];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        q[j] = ld_codes<VEC>(codes + (t * 4 + j) * C + c * VEC);
        e[j] = __ldg(scales + (t * 4 + j) * nb + c * VEC / kBlock);
      }
      load_f32<VEC>(go + t * C + c * VEC, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float f[VEC];
        restore<FMT, VEC>(q[j], scale_value(e[j]), f);
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[j] = fmaf(f[k], g[k], acc[j]);
      }
    }
    warp_reduce_scatter<4>(acc, lane);
    if ((lane & 7) == 0) __stcs(gh + t * 4 + scatter_index<4>(lane), acc[0]);
  }
}

// --------------------------------------------------------------- K4 backward
//   grad_lo[t,c]  = bf16( sum_i h_post[t,i] go[t,i,c] )
//   grad_hp[t,i]  = sum_c go[t,i,c] lo8[t,c]
//   grad_H[t,i,j] = sum_c go[t,i,c] x8[t,j,c]
template <int FMT, int VEC>
__global__ void __launch_bounds__(kThreads)
k4_bwd_q8_kernel(const bf16 *__restrict__ go, const uint8_t *__restrict__ xc,
                 const uint8_t *__restrict__ xs, const uint8_t *__restrict__ lc,
                 const uint8_t *__restrict__ ls, const float4 *__restrict__ hpost,
                 bf16 *__restrict__ glo, float *__restrict__ gH, float *__restrict__ ghp,
                 int64_t T, int C) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  const int nchunk = C / VEC, nb = (C + kBlock - 1) / kBlock;
  for (int64_t t = warp; t < T; t += nwarps) {
    const float4 hp4 = __ldg(hpost + t);
    const float hp[4] = {hp4.x, hp4.y, hp4.z, hp4.w};
    float accH[16], accP[4];
#pragma unroll
    for (int k = 0; k < 16; ++k) accH[k] = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) accP[k] = 0.f;
    for (int c = lane; c < nchunk; c += 32) {
      Codes<VEC> q[5];
      uint32_t e[5];
      float g[4][VEC];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        q[j] = ld_codes<VEC>(xc + (t * 4 + j) * C + c * VEC);
        e[j] = __ldg(xs + (t * 4 + j) * nb + c * VEC / kBlock);
      }
      q[4] = ld_codes<VEC>(lc + t * C + c * VEC);
      e[4] = __ldg(ls + t * nb + c * VEC / kBlock);
#pragma unroll
      for (int i = 0; i < 4; ++i) load_f32<VEC>(go + (t * 4 + i) * C + c * VEC, g[i]);
      float f[VEC], o[VEC];
      restore<FMT, VEC>(q[4], scale_value(e[4]), f);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        float s = hp[0] * g[0][k];
        s = fmaf(hp[1], g[1][k], s);
        s = fmaf(hp[2], g[2][k], s);
        o[k] = fmaf(hp[3], g[3][k], s);
#pragma unroll
        for (int i = 0; i < 4; ++i) accP[i] = fmaf(g[i][k], f[k], accP[i]);
      }
      if constexpr (VEC == 8) st8(glo + t * C + c * 8, o);
      else glo[t * C + c] = __float2bfloat16_rn(o[0]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        restore<FMT, VEC>(q[j], scale_value(e[j]), f);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
#pragma unroll
          for (int i = 0; i < 4; ++i) accH[i * 4 + j] = fmaf(g[i][k], f[k], accH[i * 4 + j]);
        }
      }
    }
    warp_reduce_scatter<16>(accH, lane);
    warp_reduce_scatter<4>(accP, lane);
    if ((lane & 1) == 0) __stcs(gH + t * 16 + scatter_index<16>(lane), accH[0]);
    if ((lane & 7) == 0) __stcs(ghp + t * 4 + scatter_index<4>(lane), accP[0]);
  }
}

}  // namespace

// The forwards take C % 8 == 0 and 16-byte aligned rows; for anything else the
// caller runs the bf16 kernel and launch_act_quantize.
void launch_k3_fwd_q8(const void *x, const float *hp, void *out, void *codes, void *scales, int fmt,
                      int64_t T, int C, cudaStream_t s) {
  FMHC_DISPATCH_FMT(fmt, {
    auto k = k3_fwd_q8_kernel<FMT>;
    launch(k, dim3(grid_for(k, T, kThreads)), dim3(kThreads), 0, s, (const bf16 *)x,
           (const float4 *)hp, (bf16 *)out, (uint8_t *)codes, (uint8_t *)scales, T, C);
  });
}

void launch_k4_fwd_q8(const void *x, const void *lo, const float *H, const float *hp, void *out,
                      void *codes, void *scales, int fmt, int64_t T, int C, cudaStream_t s) {
  FMHC_DISPATCH_FMT(fmt, {
    auto k = k4_fwd_q8_kernel<FMT>;
    launch(k, dim3(grid_for(k, T, kThreads)), dim3(kThreads), 0, s, (const bf16 *)x,
           (const bf16 *)lo, (const float4 *)H, (const float4 *)hp, (bf16 *)out, (uint8_t *)codes,
           (uint8_t *)scales, T, C);
  });
}

// vec: 8 (C % 8 == 0, bf16 rows 16-byte and code rows 8-byte aligned) or 1.
void launch_k3_bwd_q8(const void *go, const void *codes, const void *scales, int fmt, float *gh,
                      int64_t T, int C, int vec, cudaStream_t s) {
  FMHC_DISPATCH_FMT(fmt, {
    auto k = vec == 8 ? k3_bwd_q8_kernel<FMT, 8> : k3_bwd_q8_kernel<FMT, 1>;
    launch(k, dim3(grid_for(k, T, kThreads)), dim3(kThreads), 0, s, (const bf16 *)go,
           (const uint8_t *)codes, (const uint8_t *)scales, gh, T, C);
  });
}

void launch_k4_bwd_q8(const void *go, const void *xc, const void *xs, const void *lc,
                      const void *ls, int fmt, const float *hp, void *glo, float *gH, float *ghp,
                      int64_t T, int C, int vec, cudaStream_t s) {
  FMHC_DISPATCH_FMT(fmt, {
    auto k = vec == 8 ? k4_bwd_q8_kernel<FMT, 8> : k4_bwd_q8_kernel<FMT, 1>;
    launch(k, dim3(grid_for(k, T, kThreads)), dim3(kThreads), 0, s, (const bf16 *)go,
           (const uint8_t *)xc, (const uint8_t *)xs, (const uint8_t *)lc, (const uint8_t *)ls,
           (const float4 *)hp, (bf16 *)glo, gH, ghp, T, C);
  });
}

}  // namespace fmhc
