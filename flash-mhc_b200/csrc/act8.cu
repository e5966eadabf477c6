// 8-bit activation checkpoints on their own: quantise and restore (rows, C)
// tensors of bf16, f16 or f32 (format: act8.cuh).
#include "act8.cuh"
#include "fmhc_launch.h"
#include "grid.cuh"

namespace fmhc {

using namespace act8;

namespace {

constexpr int kThreads = 256;
// Chunks of eight values in flight per thread (262144 x 1024 bf16 int8 / 262144 x
// 2048 e4m3, us: quantise 8 128 / 251, 4 128 / 277, 2 134 / 273; restore 2 140 /
// 269, 4 141 / 282, 16 140 / 278).
constexpr int kRestoreUnroll = 2;
// Quantising, rows with a shorter last block keep too many places for more than two
// (262144 x 1000 / x 2040 int8, us: 2 143 / 280, 4 170 / 339, 8 190 / 388).
template <bool FLAT> constexpr int kUnroll = FLAT ? 8 : 2;

// Rows of C values (C % 8 == 0, 16-byte aligned rows) are seen as 4 * nb
// chunks of eight, nb = ceil(C / 32) blocks; chunks past C are empty.  Chunk i
// belongs to block i / 4 of the whole tensor, so four neighbouring lanes find
// their block's maximum with two shuffles.  FLAT (C % 32 == 0): no empty
// chunks, and the chunk's place is 8 i without a division.
//
// Places of this thread's N chunks from chunk i on, kThreads apart: one division,
// then additions (262144 x 1000 int8: 143 us; with a division per chunk 154-160).
template <int N, bool FLAT>
struct ChunkPlaces {
  int64_t at[N];
  bool in[N];
  __device__ __forceinline__ ChunkPlaces(int64_t i, int64_t chunks, int C, int nb4) {
    if constexpr (FLAT) {
#pragma unroll
      for (int u = 0; u < N; ++u) {
        in[u] = i + u * kThreads < chunks;
        at[u] = (i + u * kThreads) * 8;
      }
    } else {
      int64_t row = i / nb4;
      int k = int(i - row * nb4);
      const int rows = kThreads / nb4, rest = kThreads - rows * nb4;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        in[u] = i + u * kThreads < chunks && k * 8 < C;
        at[u] = row * C + k * 8;
        k += rest;
        row += rows;
        if (k >= nb4) {
          k -= nb4;
          ++row;
        }
      }
    }
  }
};

template <class E, int FMT, bool FLAT>
__global__ void __launch_bounds__(kThreads)
quantize_kernel(const E *__restrict__ x, uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                int64_t chunks, int C, int nb4) {
  constexpr int U = kUnroll<FLAT>;
  pdl_wait();
  const int64_t step = int64_t(gridDim.x) * kThreads * U;
  for (int64_t i0 = int64_t(blockIdx.x) * kThreads * U; i0 < chunks; i0 += step) {
    typename Elem<E>::Raw raw[U];
    const ChunkPlaces<U, FLAT> p(i0 + threadIdx.x, chunks, C, nb4);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      raw[u] = {};
      if (p.in[u]) raw[u] = ld8(x + p.at[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * kThreads + threadIdx.x;
      float f[8];
      Elem<E>::widen(raw[u], f);
      const uint32_t e = scale_byte<FMT>(amax_block(amax8_raw<E>(raw[u])));
      if (p.in[u]) __stcs(reinterpret_cast<uint2 *>(codes + p.at[u]), encode8<FMT>(f, e));
      if ((threadIdx.x & 3) == 0 && i < chunks) __stcs(scales + (i >> 2), uint8_t(e));
    }
  }
}

template <class E, int FMT, bool FLAT>
__global__ void __launch_bounds__(kThreads)
dequantize_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                  E *__restrict__ x, int64_t chunks, int C, int nb4) {
  pdl_wait();
  const int64_t step = int64_t(gridDim.x) * kThreads * kRestoreUnroll;
  for (int64_t i0 = int64_t(blockIdx.x) * kThreads * kRestoreUnroll; i0 < chunks; i0 += step) {
    uint2 raw[kRestoreUnroll];
    uint32_t e[kRestoreUnroll];
    const ChunkPlaces<kRestoreUnroll, FLAT> p(i0 + threadIdx.x, chunks, C, nb4);
#pragma unroll
    for (int u = 0; u < kRestoreUnroll; ++u) {
      if (p.in[u]) {
        raw[u] = ld_codes8(codes + p.at[u]);
        e[u] = __ldg(scales + ((i0 + u * kThreads + threadIdx.x) >> 2));
      }
    }
#pragma unroll
    for (int u = 0; u < kRestoreUnroll; ++u) {
      if (p.in[u]) {
        float f[8];
        restore<FMT>(raw[u], scale_value(e[u]), f);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = Elem<E>::fit(f[k]);
        st8(x + p.at[u], f);
      }
    }
  }
}

// Any C and any alignment: a warp takes kAnyUnroll neighbouring blocks at a time,
// one value of each per lane.
constexpr int kAnyUnroll = 8;
struct Places {  // this lane's values: where, and whether they exist
  int64_t at[kAnyUnroll];
  bool in[kAnyUnroll];
  __device__ __forceinline__ Places(int64_t b, int64_t blocks, int C, int nb, int lane) {
    const int64_t row = b / nb;
    int k = int(b - row * nb);
    const int last = C - (nb - 1) * kBlock;  // values of a row's last block
    int64_t i = row * C + k * kBlock + lane;
#pragma unroll
    for (int u = 0; u < kAnyUnroll; ++u) {
      const bool end = k + 1 == nb;
      at[u] = i;
      in[u] = b + u < blocks && (!end || lane < last);
      i += end ? last : kBlock;
      k = end ? 0 : k + 1;
    }
  }
};

template <class E, int FMT>
__global__ void __launch_bounds__(kThreads)
quantize_any_kernel(const E *__restrict__ x, uint8_t *__restrict__ codes,
                    uint8_t *__restrict__ scales, int64_t blocks, int C, int nb) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  for (int64_t b = warp * kAnyUnroll; b < blocks; b += nwarps * kAnyUnroll) {
    const Places p(b, blocks, C, nb, lane);
    E raw[kAnyUnroll];
#pragma unroll
    for (int u = 0; u < kAnyUnroll; ++u)
      if (p.in[u]) raw[u] = x[p.at[u]];
    uint32_t mine = 0;  // lane u's: the scale byte of block u
#pragma unroll
    for (int u = 0; u < kAnyUnroll; ++u) {
      const float v = p.in[u] ? Elem<E>::widen1(raw[u]) : 0.f;
      const uint32_t e = scale_byte<FMT>(
          __reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
      if (p.in[u]) codes[p.at[u]] = encode1<FMT>(v, e);
      if (lane == u) mine = e;
    }
    if (lane < kAnyUnroll && b + lane < blocks) scales[b + lane] = uint8_t(mine);
  }
}

template <class E, int FMT>
__global__ void __launch_bounds__(kThreads)
dequantize_any_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                      E *__restrict__ x, int64_t blocks, int C, int nb) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  for (int64_t b = warp * kAnyUnroll; b < blocks; b += nwarps * kAnyUnroll) {
    const Places p(b, blocks, C, nb, lane);
    uint8_t raw[kAnyUnroll], e[kAnyUnroll];
#pragma unroll
    for (int u = 0; u < kAnyUnroll; ++u)
      if (p.in[u]) {
        raw[u] = codes[p.at[u]];
        e[u] = scales[b + u];
      }
#pragma unroll
    for (int u = 0; u < kAnyUnroll; ++u)
      if (p.in[u])
        x[p.at[u]] = Elem<E>::narrow1(Elem<E>::fit(decode1<FMT>(raw[u]) * scale_value(e[u])));
  }
}

template <class E, int FMT>
void quantize(const void *x, void *codes, void *scales, int64_t rows, int C, bool vec,
              cudaStream_t s) {
  const int nb = (C + kBlock - 1) / kBlock;
  if (vec) {
    const int per_warp = 32 * (C % kBlock ? kUnroll<false> : kUnroll<true>);
    const int64_t chunks = rows * nb * 4, warps = (chunks + per_warp - 1) / per_warp;
    auto k = C % kBlock ? quantize_kernel<E, FMT, false> : quantize_kernel<E, FMT, true>;
    launch(k, dim3(grid_for(k, warps, kThreads)), dim3(kThreads), 0, s, (const E *)x,
           (uint8_t *)codes, (uint8_t *)scales, chunks, C, 4 * nb);
  } else {
    auto k = quantize_any_kernel<E, FMT>;
    launch(k, dim3(grid_for(k, (rows * nb + kAnyUnroll - 1) / kAnyUnroll, kThreads)), dim3(kThreads), 0, s, (const E *)x,
           (uint8_t *)codes, (uint8_t *)scales, rows * nb, C, nb);
  }
}

template <class E, int FMT>
void dequantize(const void *codes, const void *scales, void *x, int64_t rows, int C, bool vec,
                cudaStream_t s) {
  const int nb = (C + kBlock - 1) / kBlock;
  if (vec) {
    const int64_t chunks = rows * nb * 4, warps = (chunks + 32 * kRestoreUnroll - 1) / (32 * kRestoreUnroll);
    auto k = C % kBlock ? dequantize_kernel<E, FMT, false> : dequantize_kernel<E, FMT, true>;
    launch(k, dim3(grid_for(k, warps, kThreads)), dim3(kThreads), 0, s, (const uint8_t *)codes,
           (const uint8_t *)scales, (E *)x, chunks, C, 4 * nb);
  } else {
    auto k = dequantize_any_kernel<E, FMT>;
    launch(k, dim3(grid_for(k, (rows * nb + kAnyUnroll - 1) / kAnyUnroll, kThreads)), dim3(kThreads), 0, s, (const uint8_t *)codes,
           (const uint8_t *)scales, (E *)x, rows * nb, C, nb);
  }
}

}  // namespace

void launch_act_quantize(const void *x, int dtype, void *codes, int fmt, void *scales, int64_t rows,
                         int C, bool vec, cudaStream_t s) {
  FMHC_DISPATCH_ELEM(dtype, FMHC_DISPATCH_FMT(fmt, quantize<E, FMT>(x, codes, scales, rows, C, vec, s)));
}

void launch_act_dequantize(const void *codes, int fmt, const void *scales, void *x, int dtype,
                           int64_t rows, int C, bool vec, cudaStream_t s) {
  FMHC_DISPATCH_ELEM(dtype, FMHC_DISPATCH_FMT(fmt, dequantize<E, FMT>(codes, scales, x, rows, C, vec, s)));
}

}  // namespace fmhc
