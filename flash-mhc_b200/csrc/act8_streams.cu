// The stream mixings K3 and K4 with 8-bit activation checkpoints (format:
// act8.cuh): the forwards that also write the codes of what they read, and the
// backwards that read codes where k3k4_stream.cu reads bf16.
//
// Work mapping as in k3k4_stream.cu: one warp per token, lanes walk C in chunks
// of eight values.  Four neighbouring lanes hold one block of 32 values, so a
// block's maximum takes two shuffles, and lane 4k writes or reads its scale.
//
// The backwards read less per lane and iteration than the bf16 kernels (codes
// are half as wide) and need the registers for their sums, so loads into
// registers leave too few bytes in flight: a first version, shaped like the bf16
// kernels, reached 0.56-0.66 of the copy rate.  They prefetch through a
// shared-memory ring instead (lane_ring.cuh), one block per SM, and reach
// 0.85-0.97 (T = 65536, C = 1024 int8 / C = 2048 e4m3: K3 74 / 131 us, K4 163 /
// 321).  Scale bytes and h_post are loaded a step ahead into registers; through
// the ring, too, they cost more copies than they hid (K3 83 / 143).
#include "act8.cuh"
#include "fmhc_launch.h"
#include "grid.cuh"
#include "lane_ring.cuh"

namespace fmhc {

using namespace act8;
using bf16 = __nv_bfloat16;

namespace {

constexpr int kThreads = 256;

// Position of a warp's pipeline: token t, and this lane's chunk of eight values.
struct Cursor {
  int64_t t;
  int c;
};
__device__ __forceinline__ void advance(Cursor &p, int lane, int nchunk, int64_t nwarps) {
  p.c += 32;
  if (p.c - lane >= nchunk) {
    p.c = lane;
    p.t += nwarps;
  }
}

// ---------------------------------------------------------------- K3 forward
//   out[t,c] = bf16( sum_j h_pre[t,j] x[t,j,c] ), and x in 8 bits.
// Chunks per lane in flight and resident blocks per SM, measured at T = 65536
// (C = 1024 int8 / C = 2048 e4m3, us): 2 and 3 158 / 318; 1: 200 / 387; 2 and 4:
// 173 / 343; 4: 225 / 437; 2 with 2 blocks: 172 / 334; a shared-memory ring as
// in the backwards 158 / 350.
constexpr int kF3U = 2, kF3Blocks = 3;
template <int FMT>
__global__ void __launch_bounds__(kThreads, kF3Blocks)
k3_fwd_q8_kernel(const bf16 *__restrict__ x, const float4 *__restrict__ hp, bf16 *__restrict__ out,
                 uint8_t *__restrict__ codes, uint8_t *__restrict__ scales, int64_t T, int C) {
  constexpr int U = kF3U;
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  const int nchunk = C / 8, nb = (C + kBlock - 1) / kBlock;
  for (int64_t t = warp; t < T; t += nwarps) {
    const float4 h = __ldg(hp + t);
    const float hj[4] = {h.x, h.y, h.z, h.w};
    const bf16 *xr = x + t * 4 * C;
    for (int c0 = 0; c0 < nchunk; c0 += 32 * U) {
      uint4 a[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + 32 * u + lane;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          a[u][j] = make_uint4(0, 0, 0, 0);
          if (c < nchunk) a[u][j] = ld8(xr + j * C + c * 8);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + 32 * u + lane;
        if (c - lane >= nchunk) break;  // the whole warp is past the row
        const bool in = c < nchunk;
        float o[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float f[8];
          Elem<bf16>::widen(a[u][j], f);
#pragma unroll
          for (int k = 0; k < 8; ++k) o[k] = j ? fmaf(hj[j], f[k], o[k]) : hj[0] * f[k];
          const uint32_t e = scale_byte<FMT>(amax_block(amax8_raw<bf16>(a[u][j])));
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
}

// ---------------------------------------------------------------- K4 forward
//   out[t,i,c] = bf16( sum_j H[t,i,j] x[t,j,c] + h_post[t,i] lo[t,c] ), and lo
//   in 8 bits.
// Chunks per lane in flight and resident blocks per SM, as above: 2 and 2 208 /
// 408 us; 4 and 1: 211 / 403; 1 and 2: 224 / 438; 2 and 1: 245 / 474; a ring:
// 224 / 434.
constexpr int kF4U = 2, kF4Blocks = 2;
template <int FMT>
__global__ void __launch_bounds__(kThreads, kF4Blocks)
k4_fwd_q8_kernel(const bf16 *__restrict__ x, const bf16 *__restrict__ lo,
                 const float4 *__restrict__ H, const float4 *__restrict__ hpost,
                 bf16 *__restrict__ out, uint8_t *__restrict__ codes,
                 uint8_t *__restrict__ scales, int64_t T, int C) {
  constexpr int U = kF4U;
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
    for (int c0 = 0; c0 < nchunk; c0 += 32 * U) {
      uint4 a[U][4], l[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + 32 * u + lane;
        l[u] = make_uint4(0, 0, 0, 0);
        if (c < nchunk) {
          l[u] = ld8(lo + t * C + c * 8);
#pragma unroll
          for (int j = 0; j < 4; ++j) a[u][j] = ld8(xr + j * C + c * 8);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = c0 + 32 * u + lane;
        if (c - lane >= nchunk) break;  // the whole warp is past the row
        float fl[8];
        Elem<bf16>::widen(l[u], fl);
        const uint32_t e = scale_byte<FMT>(amax_block(amax8_raw<bf16>(l[u])));
        if (c < nchunk) {
          float fx[4][8];
#pragma unroll
          for (int j = 0; j < 4; ++j) Elem<bf16>::widen(a[u][j], fx[j]);
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
}

// --------------------------------------------------------- backward rings
// warp_reduce_scatter with its choices between values.  There, `upper ? v[k] :
// v[k + half]` chooses between addresses and puts v into local memory, which cost
// K4's backward 26 of 189 us here; the bf16 kernel is short of registers and
// faster with it (305 against 328 us).
template <int N>
__device__ __forceinline__ void reduce_scatter(float (&v)[N], int lane) {
  int live = N;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    if (live > 1) {
      const int half = live >> 1;
      const bool upper = (lane & off) != 0;
#pragma unroll
      for (int k = 0; k < half; ++k) {
        const float a = v[k], b = v[k + half];
        const float send = upper ? a : b, keep = upper ? b : a;
        v[k] = keep + __shfl_xor_sync(0xffffffffu, send, off);
      }
      live = half;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
    }
  }
}

// Eight codes, scaled.
template <int FMT>
__device__ __forceinline__ void restore8(uint2 q, uint32_t e, float2 (&f)[4]) {
  decode4x2<FMT>(q.x, f[0], f[1]);
  decode4x2<FMT>(q.y, f[2], f[3]);
  const float2 s = both(scale_value(e));
#pragma unroll
  for (int k = 0; k < 4; ++k) f[k] = mul2(f[k], s);
}
__device__ __forceinline__ void widen8(uint4 r, float2 (&f)[4]) {
  f[0] = make_float2(bf16lo(r.x), bf16hi(r.x));
  f[1] = make_float2(bf16lo(r.y), bf16hi(r.y));
  f[2] = make_float2(bf16lo(r.z), bf16hi(r.z));
  f[3] = make_float2(bf16lo(r.w), bf16hi(r.w));
}

// --------------------------------------------------------------- K3 backward
//   grad_h[t,j] = sum_c x8[t,j,c] go[t,c]
constexpr int kK3Warps = 32, kK3Stages = 4;
struct K3Stage {  // of one warp
  uint4 go[32];
  uint2 x[4][32];
};
template <int FMT>
__global__ void __launch_bounds__(32 * kK3Warps, 1)
k3_bwd_q8_kernel(const bf16 *__restrict__ go, const uint8_t *__restrict__ codes,
                 const uint8_t *__restrict__ scales, float *__restrict__ gh, int64_t T, int C) {
  extern __shared__ uint4 dyn[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t nwarps = int64_t(gridDim.x) * (blockDim.x >> 5);
  const int nchunk = C / 8, nb = (C + kBlock - 1) / kBlock;
  K3Stage *ring = reinterpret_cast<K3Stage *>(dyn) + warp * kK3Stages;
  pdl_wait();
  const auto fetch = [&](const Cursor &p, int stage) {
    if (p.t < T && p.c < nchunk) {
      copy_async<16>(&ring[stage].go[lane], go + p.t * C + p.c * 8);
#pragma unroll
      for (int j = 0; j < 4; ++j) copy_async<8>(&ring[stage].x[j][lane], codes + (p.t * 4 + j) * C + p.c * 8);
    }
    copy_commit();
  };
  uint32_t e[4] = {0, 0, 0, 0};
  const auto fetch_scales = [&](const Cursor &p) {
    if (p.t < T && p.c < nchunk) {
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = __ldg(scales + (p.t * 4 + j) * nb + (p.c >> 2));
    }
  };
  Cursor now{int64_t(warp) * gridDim.x + blockIdx.x, lane}, ahead = now;
#pragma unroll
  for (int s = 0; s < kK3Stages - 1; ++s) {
    fetch(ahead, s);
    advance(ahead, lane, nchunk, nwarps);
  }
  fetch_scales(now);
  int stage = 0;
  float2 acc[4] = {both(0.f), both(0.f), both(0.f), both(0.f)};
  while (now.t < T) {
    fetch(ahead, stage == 0 ? kK3Stages - 1 : stage - 1);
    advance(ahead, lane, nchunk, nwarps);
    const uint32_t e0[4] = {e[0], e[1], e[2], e[3]};
    Cursor next = now;
    advance(next, lane, nchunk, nwarps);
    fetch_scales(next);
    copy_wait<kK3Stages - 1>();
    if (now.c < nchunk) {
      float2 g[4], f[4];
      widen8(ring[stage].go[lane], g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        restore8<FMT>(ring[stage].x[j][lane], e0[j], f);
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[j] = fma2(f[k], g[k], acc[j]);
      }
    }
    if (next.t != now.t) {  // the token's last chunks
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = acc[j].x + acc[j].y;
        acc[j] = both(0.f);
      }
      reduce_scatter<4>(v, lane);
      if ((lane & 7) == 0) __stcs(gh + now.t * 4 + scatter_index<4>(lane), v[0]);
    }
    now = next;
    if (++stage == kK3Stages) stage = 0;
  }
}

// --------------------------------------------------------------- K4 backward
//   grad_lo[t,c]  = bf16( sum_i h_post[t,i] go[t,i,c] )
//   grad_hp[t,i]  = sum_c go[t,i,c] lo8[t,c]
//   grad_H[t,i,j] = sum_c go[t,i,c] x8[t,j,c]
constexpr int kK4Warps = 16, kK4Stages = 4;
struct K4Stage {  // of one warp
  uint4 go[4][32];
  uint2 x[5][32];  // the four streams and lo
};
template <int FMT>
__global__ void __launch_bounds__(32 * kK4Warps, 1)
k4_bwd_q8_kernel(const bf16 *__restrict__ go, const uint8_t *__restrict__ xc,
                 const uint8_t *__restrict__ xs, const uint8_t *__restrict__ lc,
                 const uint8_t *__restrict__ ls, const float4 *__restrict__ hpost,
                 bf16 *__restrict__ glo, float *__restrict__ gH, float *__restrict__ ghp,
                 int64_t T, int C) {
  extern __shared__ uint4 dyn[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t nwarps = int64_t(gridDim.x) * (blockDim.x >> 5);
  const int nchunk = C / 8, nb = (C + kBlock - 1) / kBlock;
  K4Stage *ring = reinterpret_cast<K4Stage *>(dyn) + warp * kK4Stages;
  pdl_wait();
  const auto fetch = [&](const Cursor &p, int stage) {
    if (p.t < T && p.c < nchunk) {
#pragma unroll
      for (int i = 0; i < 4; ++i) copy_async<16>(&ring[stage].go[i][lane], go + (p.t * 4 + i) * C + p.c * 8);
#pragma unroll
      for (int j = 0; j < 4; ++j) copy_async<8>(&ring[stage].x[j][lane], xc + (p.t * 4 + j) * C + p.c * 8);
      copy_async<8>(&ring[stage].x[4][lane], lc + p.t * C + p.c * 8);
    }
    copy_commit();
  };
  uint32_t e[5] = {0, 0, 0, 0, 0};
  float4 hp = make_float4(0.f, 0.f, 0.f, 0.f);
  const auto fetch_scales = [&](const Cursor &p) {
    if (p.t < T) {
      hp = __ldg(hpost + p.t);
      if (p.c < nchunk) {
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = __ldg(xs + (p.t * 4 + j) * nb + (p.c >> 2));
        e[4] = __ldg(ls + p.t * nb + (p.c >> 2));
      }
    }
  };
  Cursor now{int64_t(warp) * gridDim.x + blockIdx.x, lane}, ahead = now;
#pragma unroll
  for (int s = 0; s < kK4Stages - 1; ++s) {
    fetch(ahead, s);
    advance(ahead, lane, nchunk, nwarps);
  }
  fetch_scales(now);
  int stage = 0;
  float2 accH[4][4], accP[4];  // of even and odd columns
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    accP[i] = both(0.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) accH[i][j] = both(0.f);
  }
  while (now.t < T) {
    fetch(ahead, stage == 0 ? kK4Stages - 1 : stage - 1);
    advance(ahead, lane, nchunk, nwarps);
    const uint32_t e0[5] = {e[0], e[1], e[2], e[3], e[4]};
    const float4 h = hp;
    Cursor next = now;
    advance(next, lane, nchunk, nwarps);
    fetch_scales(next);
    copy_wait<kK4Stages - 1>();
    if (now.c < nchunk) {
      float2 g[4][4], f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) widen8(ring[stage].go[i][lane], g[i]);
      restore8<FMT>(ring[stage].x[4][lane], e0[4], f);
      float o[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float2 s = mul2(both(h.x), g[0][k]);  // in the order of fmhc_k4_bwd
        s = fma2(both(h.y), g[1][k], s);
        s = fma2(both(h.z), g[2][k], s);
        s = fma2(both(h.w), g[3][k], s);
        o[2 * k] = s.x;
        o[2 * k + 1] = s.y;
#pragma unroll
        for (int i = 0; i < 4; ++i) accP[i] = fma2(g[i][k], f[k], accP[i]);
      }
      st8(glo + now.t * C + now.c * 8, o);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        restore8<FMT>(ring[stage].x[j][lane], e0[j], f);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) accH[i][j] = fma2(g[i][k], f[k], accH[i][j]);
      }
    }
    if (next.t != now.t) {  // the token's last chunks
      float v[16], w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = accP[i].x + accP[i].y;
        accP[i] = both(0.f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[i * 4 + j] = accH[i][j].x + accH[i][j].y;
          accH[i][j] = both(0.f);
        }
      }
      reduce_scatter<16>(v, lane);
      reduce_scatter<4>(w, lane);
      if ((lane & 1) == 0) __stcs(gH + now.t * 16 + scatter_index<16>(lane), v[0]);
      if ((lane & 7) == 0) __stcs(ghp + now.t * 4 + scatter_index<4>(lane), w[0]);
    }
    now = next;
    if (++stage == kK4Stages) stage = 0;
  }
}

// ---------------------------------------------- any width and any alignment
// One warp per token, one value per lane and load: the rows of a token start at
// different places in a word.
template <int FMT>
__global__ void __launch_bounds__(kThreads)
k3_bwd_q8_any_kernel(const bf16 *__restrict__ go, const uint8_t *__restrict__ codes,
                     const uint8_t *__restrict__ scales, float *__restrict__ gh, int64_t T, int C) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  const int nb = (C + kBlock - 1) / kBlock;
  for (int64_t t = warp; t < T; t += nwarps) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c = lane; c < C; c += 32) {
      const float g = Elem<bf16>::widen1(go[t * C + c]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc[j] = fmaf(decode1<FMT>(codes[(t * 4 + j) * C + c]) * scale_value(scales[(t * 4 + j) * nb + c / kBlock]),
                      g, acc[j]);
    }
    reduce_scatter<4>(acc, lane);
    if ((lane & 7) == 0) gh[t * 4 + scatter_index<4>(lane)] = acc[0];
  }
}

template <int FMT>
__global__ void __launch_bounds__(kThreads)
k4_bwd_q8_any_kernel(const bf16 *__restrict__ go, const uint8_t *__restrict__ xc,
                     const uint8_t *__restrict__ xs, const uint8_t *__restrict__ lc,
                     const uint8_t *__restrict__ ls, const float4 *__restrict__ hpost,
                     bf16 *__restrict__ glo, float *__restrict__ gH, float *__restrict__ ghp,
                     int64_t T, int C) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  const int nb = (C + kBlock - 1) / kBlock;
  for (int64_t t = warp; t < T; t += nwarps) {
    const float4 h = __ldg(hpost + t);
    float accH[16], accP[4];
#pragma unroll
    for (int k = 0; k < 16; ++k) accH[k] = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) accP[k] = 0.f;
    const bf16 *gr = go + t * 4 * C;
    const uint8_t *xr = xc + t * 4 * C, *sr = xs + t * 4 * nb, *lr = lc + t * C, *lsr = ls + t * nb;
    // All of a step's loads first, one step at a time: 520 / 503 us (int8 / e4m3) at T
    // = 65536, C = 1023; as the compiler unrolls it otherwise 565-1069.
#pragma unroll 1
    for (int c = lane; c < C; c += 32) {
      const int k = c / kBlock;
      bf16 raw[4];
      uint8_t x[5], e[5];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        raw[j] = gr[j * C + c];
        x[j] = xr[j * C + c];
        e[j] = sr[j * nb + k];
      }
      x[4] = lr[c];
      e[4] = lsr[k];
      float g[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = Elem<bf16>::widen1(raw[i]);
      glo[t * C + c] = __float2bfloat16_rn(fmaf(h.w, g[3], fmaf(h.z, g[2], fmaf(h.y, g[1], h.x * g[0]))));
      const float l = decode1<FMT>(x[4]) * scale_value(e[4]);
#pragma unroll
      for (int i = 0; i < 4; ++i) accP[i] = fmaf(g[i], l, accP[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float v = decode1<FMT>(x[j]) * scale_value(e[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) accH[i * 4 + j] = fmaf(g[i], v, accH[i * 4 + j]);
      }
    }
    reduce_scatter<16>(accH, lane);
    reduce_scatter<4>(accP, lane);
    if ((lane & 1) == 0) gH[t * 16 + scatter_index<16>(lane)] = accH[0];
    if ((lane & 7) == 0) ghp[t * 4 + scatter_index<4>(lane)] = accP[0];
  }
}

// Warps per block of the ring kernels: few tokens spread over the SMs, many
// fill them.
int ring_warps(int64_t T, int most) {
  const int64_t per_sm = (T + sm_count() - 1) / sm_count();
  return int(per_sm < most ? (per_sm < 1 ? 1 : per_sm) : most);
}
int ring_blocks(int64_t T, int warps) {
  const int64_t need = (T + warps - 1) / warps;
  return int(need < sm_count() ? need : sm_count());
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
    if (vec == 8) {
      const int warps = ring_warps(T, kK3Warps);
      const size_t smem = sizeof(K3Stage) * kK3Stages * warps;
      auto k = k3_bwd_q8_kernel<FMT>;
      allow_smem(reinterpret_cast<const void *>(k), smem);
      launch(k, dim3(ring_blocks(T, warps)), dim3(32 * warps), smem, s, (const bf16 *)go,
             (const uint8_t *)codes, (const uint8_t *)scales, gh, T, C);
    } else {
      auto k = k3_bwd_q8_any_kernel<FMT>;
      launch(k, dim3(grid_for(k, T, kThreads)), dim3(kThreads), 0, s, (const bf16 *)go,
             (const uint8_t *)codes, (const uint8_t *)scales, gh, T, C);
    }
  });
}

void launch_k4_bwd_q8(const void *go, const void *xc, const void *xs, const void *lc,
                      const void *ls, int fmt, const float *hp, void *glo, float *gH, float *ghp,
                      int64_t T, int C, int vec, cudaStream_t s) {
  FMHC_DISPATCH_FMT(fmt, {
    if (vec == 8) {
      const int warps = ring_warps(T, kK4Warps);
      const size_t smem = sizeof(K4Stage) * kK4Stages * warps;
      auto k = k4_bwd_q8_kernel<FMT>;
      allow_smem(reinterpret_cast<const void *>(k), smem);
      launch(k, dim3(ring_blocks(T, warps)), dim3(32 * warps), smem, s, (const bf16 *)go,
             (const uint8_t *)xc, (const uint8_t *)xs, (const uint8_t *)lc, (const uint8_t *)ls,
             (const float4 *)hp, (bf16 *)glo, gH, ghp, T, C);
    } else {
      auto k = k4_bwd_q8_any_kernel<FMT>;
      launch(k, dim3(grid_for(k, T, kThreads)), dim3(kThreads), 0, s, (const bf16 *)go,
             (const uint8_t *)xc, (const uint8_t *)xs, (const uint8_t *)lc, (const uint8_t *)ls,
             (const float4 *)hp, (bf16 *)glo, gH, ghp, T, C);
    }
  });
}

}  // namespace fmhc
