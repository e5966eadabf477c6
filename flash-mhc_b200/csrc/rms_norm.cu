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
#include "fmhc_launch.h"
#include "norm_rows.cuh"
#include "rows8.cuh"

namespace fmhc {

using namespace act8;
using namespace norm_rows;

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxParts = 1024;

// ---------------------------------------------- any width and any alignment
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
// partials.
int any_slices(int64_t rows, int C) {
  if (rows <= 128) return 1;
  const int64_t cols = (C + 31) / 32;
  int64_t n = (8 * int64_t(sm_count()) + cols - 1) / cols;
  n = std::min<int64_t>(n, (rows + 31) / 32);
  return int(std::min<int64_t>(std::max<int64_t>(n, 1), kMaxParts));
}

}  // namespace

void launch_rms_fwd(const void *x, int dtype, const void *res, const void *w, int pdt, float eps,
                    void *y, void *total, float *rstd, void *codes, int64_t stride, float *scales,
                    int64_t rows, int C, cudaStream_t s) {
  FMHC_DISPATCH_ELEM(dtype, {
    auto k = codes != nullptr ? rms_fwd_any_kernel<E, true> : rms_fwd_any_kernel<E, false>;
    launch(k, dim3(grid_for(k, rows * kWarps, kThreads)), dim3(kThreads), 0, s, (const E *)x,
           (const E *)res, w, pdt, eps, (E *)y, (E *)total, rstd, (int8_t *)codes, stride, scales, rows, C);
  });
}

int64_t rms_bwd_workspace_bytes(int64_t rows, int C) {
  if (rows < 1 || C < 1) return 0;
  return (int64_t(any_slices(rows, C)) * C * 4 + 255) & ~int64_t(255);
}

void launch_rms_bwd(const void *g, int dtype, const void *gt, const void *x, const float *rstd,
                    const void *w, int pdt, void *gx, void *gw, float *ws, int64_t rows, int C,
                    cudaStream_t s) {
  FMHC_DISPATCH_ELEM(dtype, {
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
