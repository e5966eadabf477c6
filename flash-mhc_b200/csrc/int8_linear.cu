// Linear layer from 8-bit rows (rows8.cuh):
//
//   y[t, n] = (xs[t] ws[n]) sum_k xc[t, k] wc[n, k] + b[n],  rounded once
//
// The sum of products is a whole number and exact (K < 2^17 keeps it within 32
// bits); the product of the two scales is taken first, in f32.
#include "act8.cuh"
#include "fmhc_launch.h"
#include "rows8.cuh"

namespace fmhc {

using namespace act8;

namespace {

__device__ __forceinline__ float bias1(const void *b, int dtype, int64_t n) {
  if (b == nullptr) return 0.f;
  if (dtype == 0) return reinterpret_cast<const float *>(b)[n];
  if (dtype == 1) return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(b)[n]);
  return __half2float(reinterpret_cast<const __half *>(b)[n]);
}

// A 32 x 32 tile of y per block of 256 threads; 64 columns of K at a time.
template <class E>
__global__ void __launch_bounds__(256)
int8_linear_tile_kernel(const int8_t *__restrict__ xc, int64_t xstride, const float *__restrict__ xs,
                        const int8_t *__restrict__ wc, int64_t wstride, const float *__restrict__ ws,
                        const void *__restrict__ b, int bdt, E *__restrict__ y, int64_t T, int64_t N, int K) {
  __shared__ int xt[32][17], wt[32][17];
  pdl_wait();
  const int64_t n0 = int64_t(blockIdx.x) * 32;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int64_t t0 = int64_t(blockIdx.y) * 32; t0 < T; t0 += int64_t(gridDim.y) * 32) {
    int acc[4] = {0, 0, 0, 0};
    for (int k0 = 0; k0 < K; k0 += 64) {
      __syncthreads();
      for (int i = threadIdx.x; i < 32 * 64; i += 256) {
        const int r = i >> 6, k = i & 63;
        reinterpret_cast<int8_t *>(&xt[r][0])[k] = t0 + r < T && k0 + k < K ? xc[(t0 + r) * xstride + k0 + k] : int8_t(0);
        reinterpret_cast<int8_t *>(&wt[r][0])[k] = n0 + r < N && k0 + k < K ? wc[(n0 + r) * wstride + k0 + k] : int8_t(0);
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 16; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = __dp4a(xt[ty * 4 + i][k], wt[tx][k], acc[i]);
    }
    if (n0 + tx < N)
      for (int i = 0; i < 4; ++i) {
        const int64_t t = t0 + ty * 4 + i;
        if (t < T) y[t * N + n0 + tx] = Elem<E>::narrow1(fmaf(float(acc[i]), xs[t] * ws[n0 + tx], bias1(b, bdt, n0 + tx)));
      }
  }
}

}  // namespace

void launch_int8_linear(const void *xc, int64_t xstride, const float *xs, const void *wc, int64_t wstride,
                        const float *ws, const void *b, int bdt, void *y, int ydt, int64_t T, int64_t N,
                        int K, cudaStream_t s) {
  FMHC_DISPATCH_ELEM(ydt, {
    const int64_t rows = (T + 31) / 32;
    launch(int8_linear_tile_kernel<E>, dim3(unsigned((N + 31) / 32), unsigned(rows < 65535 ? rows : 65535)),
           dim3(256), 0, s, (const int8_t *)xc, xstride, xs, (const int8_t *)wc, wstride, ws, b, bdt,
           (E *)y, T, N, K);
  });
}

}  // namespace fmhc
