// Rows put into 8 bits and restored (format: rows8.cuh).
#include "act8.cuh"
#include "fmhc_launch.h"
#include "grid.cuh"
#include "rows8.cuh"

namespace fmhc {

using namespace act8;

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

template <class E>
__global__ void __launch_bounds__(kThreads)
row_quantize_any_kernel(const E *__restrict__ x, int8_t *__restrict__ codes, int64_t stride,
                        float *__restrict__ scales, int64_t rows, int C) {
  __shared__ uint32_t sh[kWarps];
  pdl_wait();
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    uint32_t m = 0;
    for (int c = threadIdx.x; c < C; c += kThreads) m = max(m, rows8::magnitude(Elem<E>::widen1(x[r * C + c])));
    m = __reduce_max_sync(0xffffffffu, m);
    __syncthreads();  // the previous row's reads are over
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) m = max(m, sh[i]);
    const rows8::RowScale q = rows8::row_scale(m);
    if (threadIdx.x == 0) scales[r] = q.scale;
    for (int c = threadIdx.x; c < C; c += kThreads)
      codes[r * stride + c] = rows8::code1(Elem<E>::widen1(x[r * C + c]), q.inv);
  }
}

template <class E>
__global__ void __launch_bounds__(kThreads)
row_dequantize_any_kernel(const int8_t *__restrict__ codes, int64_t stride, const float *__restrict__ scales,
                          E *__restrict__ x, int64_t rows, int C) {
  pdl_wait();
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float s = scales[r];
    for (int c = threadIdx.x; c < C; c += kThreads)
      x[r * C + c] = Elem<E>::narrow1(float(codes[r * stride + c]) * s);
  }
}

}  // namespace

void launch_row_quantize(const void *x, int dtype, void *codes, int64_t stride, float *scales,
                         int64_t rows, int C, cudaStream_t s) {
  FMHC_DISPATCH_ELEM(dtype, {
    auto k = row_quantize_any_kernel<E>;
    launch(k, dim3(grid_for(k, rows * kWarps, kThreads)), dim3(kThreads), 0, s, (const E *)x,
           (int8_t *)codes, stride, scales, rows, C);
  });
}

void launch_row_dequantize(const void *codes, int64_t stride, const float *scales, void *x, int dtype,
                           int64_t rows, int C, cudaStream_t s) {
  FMHC_DISPATCH_ELEM(dtype, {
    auto k = row_dequantize_any_kernel<E>;
    launch(k, dim3(grid_for(k, rows * kWarps, kThreads)), dim3(kThreads), 0, s, (const int8_t *)codes,
           stride, scales, (E *)x, rows, C);
  });
}

}  // namespace fmhc
