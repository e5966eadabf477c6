// Root-mean-square norm over rows of C values, forward and backward, with a
// residual's addition in front and an output in 8 bits for serving (rows8.cuh).
//
//   v     = x, or x + residual rounded to x's type (written as `total`)
//   rstd  = 1 / sqrt(<v^2> + eps)                           (<> : mean over C)
//   y     = v rstd w, rounded once, or as a row of int8 codes and a scale
//   grad_v = rstd (gw - xh <gw xh>) + grad_total,  gw = g w,  xh = v rstd
//   grad_w = sum over rows of g xh
//
// Sums are f32.  The norm is that of the rounded total, which the backward reads
// too, so forward and gradients belong to the same values.
//
// Memory bounds them.  Measured, bf16, us (floor of the bytes at the copy rate): norm
// 65536 x 2048 93 (83), 16384 x 8192 85 (83); with a residual 131072 x 1024 183 (165),
// 32768 x 4096 163 (165); to 8 bits 65536 x 2048 72 (62), with a residual 146 (144);
// backward 65536 x 2048 128 (124), with the gradient of total 131072 x 1024 156 (165,
// part of grad_x being still in L2).  f32 65536 x 2048: 197 (165), with a residual 365
// (330), backward 252 (248).
#include "fmhc_launch.h"
#include "norm_rows.cuh"
#include "rows8.cuh"
#include "rows_general.h"

namespace fmhc {

using namespace act8;
using namespace norm_rows;

namespace {

constexpr int kFwdWarps = 24;  // per block, one block per SM
constexpr int kBwdWarps = 16;  // for 128 registers a thread
constexpr int kThreads = 256;  // of the kernels for any width
constexpr int kWarps = kThreads / 32;
constexpr int kMaxParts = 1024;

// Most chunks per lane.  With a third array (the residual, or the gradient of total) rows
// take half as many where that covers their width.
template <class E> constexpr int kMaxNV = sizeof(E) == 2 ? 4 : 2;
// Rows in flight in the ring: the one in use and the next.  A third row made most cases
// slower (us, two / three: forward with a residual to 8 bits 131072 x 1024 142 / 165,
// backward with a third array 157 / 175).
constexpr int kStages = 2;
// -------------------------------------------------------------------- forward
// A team of 1..16 warps holds a row, NV chunks of eight values per lane, so that
// everything is read once; the next rows are prefetched into a shared-memory ring
// (lane_ring.cuh).  RES: with a residual.  CODES: the output as codes and scales,
// which takes a second joining of the team, for the largest magnitude.
template <class E, int NV, bool RES, bool CODES>
__global__ void __launch_bounds__(32 * kFwdWarps, 1)
rms_fwd_kernel(const E *__restrict__ x, const E *__restrict__ res, const void *__restrict__ w, int pdt,
               float eps, E *__restrict__ y, E *__restrict__ total, float *__restrict__ rstd_out,
               int8_t *__restrict__ codes, int64_t stride, float *__restrict__ scales, int64_t rows,
               int C, int team) {
  using Raw = typename Elem<E>::Raw;
  constexpr int S = kStages;
  constexpr int kChunk = 32 * int(sizeof(Raw));  // a warp's chunk in the ring
  constexpr int kStage = NV * kChunk * (RES ? 2 : 1);
  extern __shared__ uint4 dyn[];
  __shared__ float sum_slots[2][kFwdWarps];
  __shared__ uint32_t max_slots[2][kFwdWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int teams = warps / team, wt = warp % team;
  const Team tm(team, warp, lane);
  const int nchunk = C / 8;
  const uint32_t ring = shared_addr(dyn) + warp * (S * kStage) + lane * int(sizeof(Raw));
  // Warp i of the team holds the NV * 32 chunks from i * NV * 32, those below
  // nchunk; this lane every 32nd, from c0: its chunk i exists if i * 32 < left.
  const int c0 = wt * NV * 32 + lane, left = nchunk - c0;
  const float inv_C = 1.f / float(C);
  const int64_t step = int64_t(gridDim.x) * teams;
  int64_t r = int64_t(blockIdx.x) * teams + warp / team;
  pdl_wait();
  // Pointers that move on by one step of rows.
  const int64_t hop = step * C;
  const E *src = x + r * C + c0 * 8;
  const E *src2 = RES ? res + r * C + c0 * 8 : nullptr;
  E *dst = CODES ? nullptr : y + r * C + c0 * 8;
  E *dst2 = RES ? total + r * C + c0 * 8 : nullptr;
  int8_t *code_dst = CODES ? codes + r * stride + c0 * 8 : nullptr;
  int64_t fetched = r;
  const auto fetch = [&](int stage) {
    if (fetched < rows) {
      const uint32_t to = ring + stage * kStage;
      unrolled<NV>([&](auto i) {
        if (i * 32 < left) {
          copy_raw<E, i * kChunk>(to, src + i * 256);
          if constexpr (RES) copy_raw<E, (NV + i) * kChunk>(to, src2 + i * 256);
        }
      });
    }
    fetched += step;
    src += hop;
    if constexpr (RES) src2 += hop;
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s);
  float4 *ws = reinterpret_cast<float4 *>(reinterpret_cast<char *>(dyn) + warps * (S * kStage));
  keep_param(ws, w, pdt, 1.f, nchunk);
  __syncthreads();
  const uint32_t w_lo = shared_addr(ws + c0), w_hi = shared_addr(ws + nchunk + c0);
  int par = 0, stage = 0;
  for (; r < rows; r += step, par ^= 1) {
    fetch(stage == 0 ? S - 1 : stage - 1);
    copy_wait<S - 1>();
    float f[NV][8];
    float q = 0.f, q1 = 0.f;
    const uint32_t from = ring + stage * kStage;
    unrolled<NV>([&](auto i) {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[i][k] = 0.f;
      if (i * 32 < left) {
        Elem<E>::widen(load_raw<E, i * kChunk>(from), f[i]);
        if constexpr (RES) {
          float g[8];
          Elem<E>::widen(load_raw<E, (NV + i) * kChunk>(from), g);
#pragma unroll
          for (int k = 0; k < 8; ++k) f[i][k] += g[k];
          const Raw sum = Elem<E>::narrow(f[i]);
          st_raw<E>(dst2 + i * 256, sum);
          Elem<E>::widen(sum, f[i]);
        }
      }
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        q = fmaf(f[i][k], f[i][k], q);
        q1 = fmaf(f[i][k + 1], f[i][k + 1], q1);
      }
    });
    if (++stage == S) stage = 0;
    const float s = team_sum1(warp_sum(q + q1), sum_slots[par], tm, warp);
    const float rstd = rsqrtf(fmaf(s, inv_C, eps));
    if constexpr (!CODES) {
      if (wt == 0 && lane == 0) rstd_out[r] = rstd;
      unrolled<NV>([&](auto i) {
        if (i * 32 < left) {
          float fw[8], o[8];
          kept_param<i>(w_lo, w_hi, fw);
#pragma unroll
          for (int k = 0; k < 8; ++k) o[k] = f[i][k] * rstd * fw[k];
          st8(dst + i * 256, o);
        }
      });
      dst += hop;
    } else {
      uint32_t m = 0;
      unrolled<NV>([&](auto i) {
        if (i * 32 < left) {
          float fw[8];
          kept_param<i>(w_lo, w_hi, fw);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            f[i][k] = f[i][k] * rstd * fw[k];  // as y: rstd w alone may leave f32's range
            m = max(m, rows8::magnitude(f[i][k]));
          }
        }
      });
      m = team_max(__reduce_max_sync(0xffffffffu, m), max_slots[par], tm, warp);
      const rows8::RowScale sc = rows8::row_scale(m);
      if (wt == 0 && lane == 0) scales[r] = sc.scale;
      unrolled<NV>([&](auto i) {
        if (i * 32 < left) rows8::store_codes8(code_dst + i * 256, f[i], sc.inv);
      });
      code_dst += step * stride;
    }
    if constexpr (RES) dst2 += hop;
  }
}

// ------------------------------------------------------------------- backward
// As the forward.  A lane keeps the same columns for every row its team takes, so its
// share of grad_w stays in registers until the end; a block writes one partial [C],
// and rms_weight_grad_kernel adds them in block order.  THIRD: with the gradient of
// total.  The second pass over a row reads the ring again, and the weight comes from
// shared memory as f32 (or, for rows whose weight does not fit there, from global
// memory) twice: holding them would pass 128 registers.
template <class E, int NV, int S, bool THIRD, bool W_SHARED>
__global__ void __launch_bounds__(32 * kBwdWarps, 1)
rms_bwd_kernel(const E *__restrict__ g, const E *__restrict__ gt, const E *__restrict__ x,
               const float *__restrict__ rstd, const void *__restrict__ w, int pdt, E *__restrict__ gx,
               float *__restrict__ part, int64_t rows, int C, int team) {
  using Raw = typename Elem<E>::Raw;
  constexpr int kChunk = 32 * int(sizeof(Raw));
  constexpr int kStage = NV * kChunk * (THIRD ? 3 : 2);
  constexpr int kRow = 16;  // rstd of the row, per warp and stage
  extern __shared__ uint4 dyn[];
  __shared__ float slots[2][kBwdWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int teams = warps / team, wt = warp % team;
  const Team tm(team, warp, lane);
  const int nchunk = C / 8;
  const uint32_t ring = shared_addr(dyn) + warp * (S * kStage) + lane * int(sizeof(Raw));
  // Copied by one lane for the whole warp, so a warp barrier stands on both sides of a
  // refill (an ordinary load in this loop would make the shared-memory loads wait for it).
  const uint32_t ring_r = shared_addr(dyn) + warps * (S * kStage) + warp * (S * kRow);
  const int c0 = wt * NV * 32 + lane, left = nchunk - c0;
  const float inv_C = 1.f / float(C);
  const int64_t step = int64_t(gridDim.x) * teams;
  int64_t r = int64_t(blockIdx.x) * teams + warp / team;
  pdl_wait();
  const int64_t hop = step * C;
  const E *g_src = g + r * C + c0 * 8, *x_src = x + r * C + c0 * 8;
  const E *t_src = THIRD ? gt + r * C + c0 * 8 : nullptr;
  E *dst = gx + r * C + c0 * 8;
  int64_t fetched = r;
  const auto fetch = [&](int stage) {
    if (fetched < rows) {
      if (lane == 0) copy_async4(ring_r + stage * kRow, rstd + fetched);
      const uint32_t to = ring + stage * kStage;
      unrolled<NV>([&](auto i) {
        if (i * 32 < left) {
          copy_raw<E, i * kChunk>(to, g_src + i * 256);
          copy_raw<E, (NV + i) * kChunk>(to, x_src + i * 256);
          if constexpr (THIRD) copy_raw<E, (2 * NV + i) * kChunk>(to, t_src + i * 256);
        }
      });
    }
    fetched += step;
    g_src += hop;
    x_src += hop;
    if constexpr (THIRD) t_src += hop;
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s);
  float4 *ws = reinterpret_cast<float4 *>(reinterpret_cast<char *>(dyn) + warps * (S * (kStage + kRow)));
  if constexpr (W_SHARED) {
    keep_param(ws, w, pdt, 1.f, nchunk);
    __syncthreads();
  }
  const uint32_t w_lo = shared_addr(ws + c0), w_hi = shared_addr(ws + nchunk + c0);
  const auto weight = [&](auto i, float2 (&f)[4]) {
    if constexpr (W_SHARED) kept_param<i>(w_lo, w_hi, f);
    else param8x2(w, pdt, c0 + i * 32, 1.f, f);
  };
  float2 dw[NV][4];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) dw[i][k] = both(0.f);
  int par = 0, stage = 0;
  for (; r < rows; r += step, par ^= 1) {
    __syncwarp();
    fetch(stage == 0 ? S - 1 : stage - 1);
    copy_wait<S - 1>();
    __syncwarp();
    const float rs = load_shared_f32(ring_r + stage * kRow);
    const uint32_t from = ring + stage * kStage;
    float2 dot = both(0.f);
    unrolled<NV>([&](auto i) {
      if (i * 32 < left) {
        float2 fg[4], fx[4], fw[4];
        widen2<E>(load_raw<E, i * kChunk>(from), fg);
        widen2<E>(load_raw<E, (NV + i) * kChunk>(from), fx);
        weight(i, fw);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 gxh = mul2(fg[k], mul2(fx[k], both(rs)));
          dw[i][k] = add2(dw[i][k], gxh);
          dot = fma2(gxh, fw[k], dot);
        }
      }
    });
    const float sum = team_sum1(warp_sum(dot.x + dot.y), slots[par], tm, warp);
    const float2 c = both(-sum * inv_C * rs);  // times x
    unrolled<NV>([&](auto i) {
      if (i * 32 < left) {
        float2 fg[4], fx[4], fw[4], ft[4];
        widen2<E>(load_raw<E, i * kChunk>(from), fg);
        widen2<E>(load_raw<E, (NV + i) * kChunk>(from), fx);
        if constexpr (THIRD) widen2<E>(load_raw<E, (2 * NV + i) * kChunk>(from), ft);
        weight(i, fw);
        float o[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 v = fma2(fx[k], c, mul2(fg[k], fw[k]));
          const float2 u = THIRD ? fma2(both(rs), v, ft[k]) : mul2(both(rs), v);
          o[2 * k] = u.x;
          o[2 * k + 1] = u.y;
        }
        st8(dst + i * 256, o);
      }
    });
    dst += hop;
    if (++stage == S) stage = 0;
  }
  if (part == nullptr) return;
  // Join the block's teams in the ring's memory (no copy is in flight: a row past the
  // end fetches nothing), in team order.
  copy_wait<0>();
  __syncthreads();
  float *sums = reinterpret_cast<float *>(dyn);  // [teams][C]
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * 32 < left) {
      float4 *to = reinterpret_cast<float4 *>(sums + (warp / team) * C + (c0 + i * 32) * 8);
      to[0] = make_float4(dw[i][0].x, dw[i][0].y, dw[i][1].x, dw[i][1].y);
      to[1] = make_float4(dw[i][2].x, dw[i][2].y, dw[i][3].x, dw[i][3].y);
    }
  __syncthreads();
  float *out = part + int64_t(blockIdx.x) * C;
  for (int c1 = threadIdx.x; c1 < C; c1 += blockDim.x) {
    float v = 0.f;
    for (int t = 0; t < teams; ++t) v += sums[t * C + c1];
    out[c1] = v;
  }
}

// ---------------------------------------------- any width and any alignment
// For pointers that are not 16-byte aligned and rows past the other kernels' widths.
// One block per row, which is read again for each step (from L1 or L2).
__device__ float block_sum(float v, float *sh) {
  v = warp_sum(v);
  __syncthreads();  // the previous use of sh is over
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) t += sh[i];
  return t;
}
__device__ uint32_t block_max(uint32_t v, uint32_t *sh) {
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) t = max(t, sh[i]);
  return t;
}

// CODES: the output as codes and scales instead of y and rstd.
template <class E, bool CODES>
__global__ void __launch_bounds__(kThreads)
rms_fwd_any_kernel(const E *__restrict__ x, const E *__restrict__ res, const void *__restrict__ w,
                   int pdt, float eps, E *__restrict__ y, E *__restrict__ total,
                   float *__restrict__ rstd_out, int8_t *__restrict__ codes, int64_t stride,
                   float *__restrict__ scales, int64_t rows, int C) {
  __shared__ float sh[kWarps];
  __shared__ uint32_t sm[kWarps];
  pdl_wait();
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const auto value = [&](int c) {
      float f = Elem<E>::widen1(x[r * C + c]);
      if (res != nullptr) f = Elem<E>::widen1(Elem<E>::narrow1(f + Elem<E>::widen1(res[r * C + c])));
      return f;
    };
    float s = 0.f;
    for (int c = threadIdx.x; c < C; c += kThreads) {
      const float f = value(c);
      if (res != nullptr) total[r * C + c] = Elem<E>::narrow1(f);
      s = fmaf(f, f, s);
    }
    const float rstd = rsqrtf(block_sum(s, sh) / float(C) + eps);
    if constexpr (!CODES) {
      if (threadIdx.x == 0) rstd_out[r] = rstd;
      for (int c = threadIdx.x; c < C; c += kThreads)
        y[r * C + c] = Elem<E>::narrow1(value(c) * rstd * param1(w, pdt, c, 1.f));
    } else {
      uint32_t m = 0;
      for (int c = threadIdx.x; c < C; c += kThreads)
        m = max(m, rows8::magnitude(value(c) * rstd * param1(w, pdt, c, 1.f)));
      const rows8::RowScale q = rows8::row_scale(block_max(m, sm));
      if (threadIdx.x == 0) scales[r] = q.scale;
      for (int c = threadIdx.x; c < C; c += kThreads)
        codes[r * stride + c] = rows8::code1(value(c) * rstd * param1(w, pdt, c, 1.f), q.inv);
    }
  }
}

template <class E>
__global__ void __launch_bounds__(kThreads)
rms_bwd_any_kernel(const E *__restrict__ g, const E *__restrict__ gt, const E *__restrict__ x,
                   const float *__restrict__ rstd, const void *__restrict__ w, int pdt,
                   E *__restrict__ gx, int64_t rows, int C) {
  __shared__ float sh[kWarps];
  pdl_wait();
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float rs = rstd[r];
    float s = 0.f;
    for (int c = threadIdx.x; c < C; c += kThreads)
      s = fmaf(Elem<E>::widen1(g[r * C + c]) * param1(w, pdt, c, 1.f), Elem<E>::widen1(x[r * C + c]) * rs, s);
    const float dot = block_sum(s, sh) / float(C);
    for (int c = threadIdx.x; c < C; c += kThreads) {
      const float gw = Elem<E>::widen1(g[r * C + c]) * param1(w, pdt, c, 1.f);
      const float xh = Elem<E>::widen1(x[r * C + c]) * rs;
      const float add = gt == nullptr ? 0.f : Elem<E>::widen1(gt[r * C + c]);
      gx[r * C + c] = Elem<E>::narrow1(fmaf(rs, fmaf(-xh, dot, gw), add));
    }
  }
}

// Partials of grad_w: block (cols of 32, slice of rows); grad_w itself if there is
// one slice.
template <class E>
__global__ void __launch_bounds__(kThreads)
rms_weight_part_any_kernel(const E *__restrict__ g, const E *__restrict__ x,
                           const float *__restrict__ rstd, float *__restrict__ part, void *gw,
                           int pdt, int64_t rows, int C) {
  __shared__ float acc[kWarps][32];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const int64_t r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
  float a = 0.f;
  if (c < C) {
#pragma unroll 4
    for (int64_t r = r0 + warp; r < r1; r += kWarps)
      a = fmaf(Elem<E>::widen1(g[r * C + c]), Elem<E>::widen1(x[r * C + c]) * rstd[r], a);
  }
  acc[warp][lane] = a;
  __syncthreads();
  if (warp == 0 && c < C) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) s += acc[i][lane];
    if (gridDim.y == 1) store_param(gw, pdt, c, s);
    else part[int64_t(blockIdx.y) * C + c] = s;
  }
}

// Adds n partials [n][C] in a fixed order: a block takes 32 columns, each of its
// 32 warps adds every 32nd partial, and the 32 results are added pairwise.
constexpr int kSumWarps = 32;
__global__ void __launch_bounds__(32 * kSumWarps)
rms_weight_grad_kernel(const float *__restrict__ part, void *__restrict__ gw, int pdt, int n, int C) {
  pdl_wait();
  __shared__ float acc[kSumWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = blockIdx.x * 32;
  float a = 0.f;
  if (c0 + lane < C) {
#pragma unroll 8
    for (int i = warp; i < n; i += kSumWarps) a += part[int64_t(i) * C + c0 + lane];
  }
  acc[warp][lane] = a;
  __syncthreads();
  const float s = warp_sum(acc[lane][warp]);
  if (lane == 0 && c0 + warp < C) store_param(gw, pdt, c0 + warp, s);
}

// Slices of 32 rows or more; up to 128 rows are one, which needs no kernel to add
// partials (as layer norm's, and measured there).
int any_slices(int64_t rows, int C) {
  if (rows <= 128) return 1;
  const int64_t cols = (C + 31) / 32;
  int64_t n = (8 * int64_t(sm_count()) + cols - 1) / cols;
  n = std::min<int64_t>(n, (rows + 31) / 32);
  return int(std::min<int64_t>(std::max<int64_t>(n, 1), kMaxParts));
}

// Rows that the kernels for any width take: not of whole chunks, or so narrow that
// several share a warp.
bool general_width(int C) { return C % 8 != 0 || C <= 128; }

// Rows over teams for the kernels above.  `half`: chunks up to half the most where
// that covers the width, and else up to the most with 16 warps.
template <class E>
bool shape_for(int64_t rows, int C, bool half, int max_warps, Shape *p) {
  if (half && register_shape(rows, C, kMaxNV<E> / 2, max_warps, p)) return true;
  return register_shape(rows, C, kMaxNV<E>, half ? 16 : max_warps, p);
}

// The forward: 16 warps, but 24 for what is bound by arithmetic: rows that go into 8 bits
// without a residual or from f32, and f32 rows on their own (us, 16 / 24: 32768 x 4096
// bf16 84 / 94, with a residual 163 / 184, both and to 8 bits 131072 x 1024 143 / 162;
// to 8 bits 65536 x 2048 82 / 72, from f32 with a residual 288 / 269, f32 207 / 197).
template <class E, bool RES, bool CODES>
bool fwd_shape(int64_t rows, int C, Shape *p) {
  constexpr bool kF32 = sizeof(E) == 4;
  return shape_for<E>(rows, C, RES, (RES ? CODES && kF32 : CODES || kF32) ? kFwdWarps : 16, p);
}
// The backward: half the chunks for 16-bit rows too (us, half / all: 65536 x 2048 bf16
// 122 / 144, 131072 x 1024 130 / 144), but not for f32 ones without a third array
// (65536 x 2048 297 / 255).
template <class E>
bool bwd_shape(int64_t rows, int C, bool third, Shape *p) {
  return shape_for<E>(rows, C, third || sizeof(E) == 2, kBwdWarps, p);
}

#define FMHC_DISPATCH_NV(NV_RT, ...)                         \
  do {                                                       \
    if ((NV_RT) == 1) { constexpr int NV = 1; __VA_ARGS__; } \
    else if ((NV_RT) == 2) { constexpr int NV = 2; __VA_ARGS__; } \
    else { constexpr int NV = kMaxNV<E>; __VA_ARGS__; }      \
  } while (0)

template <class E, bool RES, bool CODES>
bool launch_fwd(const void *x, const void *res, const void *w, int pdt, float eps, void *y, void *total,
                float *rstd, void *codes, int64_t stride, float *scales, int64_t rows, int C, cudaStream_t s) {
  Shape p;
  if (!fwd_shape<E, RES, CODES>(rows, C, &p)) return false;
  FMHC_DISPATCH_NV(p.nv, {
    auto k = rms_fwd_kernel<E, NV, RES, CODES>;
    const size_t smem = size_t(p.threads) * kStages * NV * sizeof(typename Elem<E>::Raw) * (RES ? 2 : 1) +
                        size_t(C) * 4;
    allow_smem(reinterpret_cast<const void *>(k), smem);
    launch(k, dim3(blocks_for(rows, p)), dim3(p.threads), smem, s, (const E *)x, (const E *)res, w, pdt, eps,
           (E *)y, (E *)total, rstd, (int8_t *)codes, stride, scales, rows, C, p.team);
  });
  return true;
}

template <class E, bool THIRD>
bool launch_bwd(const void *g, const void *gt, const void *x, const float *rstd, const void *w, int pdt, void *gx,
                void *gw, float *ws, int64_t rows, int C, cudaStream_t s) {
  Shape p;
  if (!bwd_shape<E>(rows, C, THIRD, &p)) return false;
  float *part = gw != nullptr ? ws : nullptr;
  const int parts = blocks_for(rows, p);
  // Three rows in flight for two arrays of wide rows (us, two / three: 32768 x 4096 134 /
  // 121, 65536 x 2048 128 / 127, 131072 x 1024 125 / 136).
  const int stages = !THIRD && p.team >= 8 ? 3 : kStages;
  FMHC_DISPATCH_NV(p.nv, {
    const size_t ring = size_t(p.threads) * stages * NV * sizeof(typename Elem<E>::Raw) * (THIRD ? 3 : 2) +
                        size_t(p.threads / 32) * stages * 16;
    // The ring's memory later holds the 32 NV bytes of sums of every thread.
    static_assert(kStages * sizeof(typename Elem<E>::Raw) * 2 >= 32, "sums fit the ring");
    const size_t with_w = ring + size_t(C) * 4;
    auto k = stages == 3 ? rms_bwd_kernel<E, NV, 3, THIRD, true> : rms_bwd_kernel<E, NV, kStages, THIRD, true>;
    size_t smem = with_w;
    if constexpr (NV == kMaxNV<E>) {
      if (with_w > kMaxSmem) {
        k = stages == 3 ? rms_bwd_kernel<E, NV, 3, THIRD, false> : rms_bwd_kernel<E, NV, kStages, THIRD, false>;
        smem = ring;
      }
    }
    allow_smem(reinterpret_cast<const void *>(k), smem);
    launch(k, dim3(parts), dim3(p.threads), smem, s, (const E *)g, (const E *)gt, (const E *)x, rstd, w, pdt,
           (E *)gx, part, rows, C, p.team);
  });
  if (part != nullptr)
    launch(rms_weight_grad_kernel, dim3((C + 31) / 32), dim3(32 * kSumWarps), 0, s, (const float *)part, gw, pdt,
           parts, C);
  return true;
}

}  // namespace

void launch_rms_fwd(const void *x, int dtype, const void *res, const void *w, int pdt, float eps,
                    void *y, void *total, float *rstd, void *codes, int64_t stride, float *scales,
                    int64_t rows, int C, bool vec, cudaStream_t s) {
  FMHC_DISPATCH_ELEM(dtype, {
    auto fast = res != nullptr ? codes != nullptr ? launch_fwd<E, true, true> : launch_fwd<E, true, false>
                               : codes != nullptr ? launch_fwd<E, false, true> : launch_fwd<E, false, false>;
    if (vec && general_width(C)) {
      if (launch_general_fwd(x, dtype, res, w, pdt, eps, y, total, rstd, codes, stride, scales, true, rows, C, s)) return;
    } else if (vec && fast(x, res, w, pdt, eps, y, total, rstd, codes, stride, scales, rows, C, s)) {
      return;
    }
    auto k = codes != nullptr ? rms_fwd_any_kernel<E, true> : rms_fwd_any_kernel<E, false>;
    launch(k, dim3(grid_for(k, rows * kWarps, kThreads)), dim3(kThreads), 0, s, (const E *)x,
           (const E *)res, w, pdt, eps, (E *)y, (E *)total, rstd, (int8_t *)codes, stride, scales, rows, C);
  });
}

int64_t rms_bwd_workspace_bytes(int64_t rows, int C) {
  if (rows < 1 || C < 1) return 0;
  // The largest of the paths, so that the size depends on neither the type nor
  // the alignment.
  int64_t n = std::max(any_slices(rows, C), general_bwd_parts(rows, C));
  Shape p;
  for (bool third : {false, true}) {
    if (bwd_shape<float>(rows, C, third, &p)) n = std::max<int64_t>(n, blocks_for(rows, p));
    if (bwd_shape<__half>(rows, C, third, &p)) n = std::max<int64_t>(n, blocks_for(rows, p));
  }
  return (n * C * 4 + 255) & ~int64_t(255);
}

void launch_rms_bwd(const void *g, int dtype, const void *gt, const void *x, const float *rstd,
                    const void *w, int pdt, void *gx, void *gw, float *ws, int64_t rows, int C,
                    bool vec, cudaStream_t s) {
  FMHC_DISPATCH_ELEM(dtype, {
    auto fast = gt != nullptr ? launch_bwd<E, true> : launch_bwd<E, false>;
    if (vec && general_width(C)) {
      if (launch_general_bwd(g, dtype, gt, x, rstd, w, pdt, gx, gw != nullptr ? ws : nullptr, rows, C, s)) {
        if (gw != nullptr)
          launch(rms_weight_grad_kernel, dim3((C + 31) / 32), dim3(32 * kSumWarps), 0, s, (const float *)ws, gw, pdt,
                 general_bwd_parts(rows, C), C);
        return;
      }
    } else if (vec && fast(g, gt, x, rstd, w, pdt, gx, gw, ws, rows, C, s)) {
      return;
    }
    auto k = rms_bwd_any_kernel<E>;
    launch(k, dim3(grid_for(k, rows * kWarps, kThreads)), dim3(kThreads), 0, s, (const E *)g,
           (const E *)gt, (const E *)x, rstd, w, pdt, (E *)gx, rows, C);
    if (gw != nullptr) {
      const int parts = any_slices(rows, C);
      launch(rms_weight_part_any_kernel<E>, dim3((C + 31) / 32, parts), dim3(kThreads), 0, s,
             (const E *)g, (const E *)x, rstd, ws, gw, pdt, rows, C);
      if (parts > 1)
        launch(rms_weight_grad_kernel, dim3((C + 31) / 32), dim3(32 * kSumWarps), 0, s,
               (const float *)ws, gw, pdt, parts, C);
    }
  });
}

}  // namespace fmhc
