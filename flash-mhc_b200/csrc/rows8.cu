// Rows put into 8 bits and restored (format: rows8.cuh).  Memory bounds both: 32768 x
// 4096 bf16 63 us and 70 us (the bytes at the copy rate take 62).  Restoring writes twice
// what it reads (to f32 four times: 65536 x 2048 159 us, 103); rows that start anywhere in
// a word restore 65536 x 1023 in 63 us (31) and 20000 x 5001 in 76 (46), bound by
// instructions.
#include "code_word.h"
#include "fmhc_launch.h"
#include "norm_rows.cuh"
#include "rows8.cuh"
#include "rows_general.h"

namespace fmhc {

using namespace act8;
using namespace norm_rows;

namespace {

// Warps per block, one block per SM, and rows in flight in the ring (us, 24 warps and
// three rows / 16 and three / 16 and two: 32768 x 4096 bf16 68 / 63 / 63, 131072 x 1024
// 68 / 67 / 61, 65536 x 2048 f32 125 / 97 / 102).
constexpr int kQuantWarps = 16;
template <class E> constexpr int kStages = sizeof(E) == 4 ? 3 : 2;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
template <class E> constexpr int kMaxNV = sizeof(E) == 2 ? 4 : 2;

// A team of warps holds a row, as in the norms (rms_norm.cu), and the next rows are
// prefetched into a shared-memory ring: x is read once.
template <class E, int NV>
__global__ void __launch_bounds__(32 * kQuantWarps, 1)
row_quantize_kernel(const E *__restrict__ x, int8_t *__restrict__ codes, int64_t stride,
                    float *__restrict__ scales, int64_t rows, int C, int team) {
  using Raw = typename Elem<E>::Raw;
  constexpr int S = kStages<E>, kChunk = 32 * int(sizeof(Raw)), kStage = NV * kChunk;
  extern __shared__ uint4 dyn[];
  __shared__ uint32_t slots[2][kQuantWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int teams = (blockDim.x >> 5) / team, wt = warp % team;
  const Team tm(team, warp, lane);
  const uint32_t ring = shared_addr(dyn) + warp * (S * kStage) + lane * int(sizeof(Raw));
  const int c0 = wt * NV * 32 + lane, left = C / 8 - c0;
  const int64_t step = int64_t(gridDim.x) * teams;
  int64_t r = int64_t(blockIdx.x) * teams + warp / team;
  pdl_wait();
  const int64_t hop = step * C;
  const E *src = x + r * C + c0 * 8;
  int8_t *dst = codes + r * stride + c0 * 8;
  int64_t fetched = r;
  const auto fetch = [&](int stage) {
    if (fetched < rows)
      unrolled<NV>([&](auto i) {
        if (i * 32 < left) copy_raw<E, i * kChunk>(ring + stage * kStage, src + i * 256);
      });
    fetched += step;
    src += hop;
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s);
  int par = 0, stage = 0;
  for (; r < rows; r += step, par ^= 1) {
    fetch(stage == 0 ? S - 1 : stage - 1);
    copy_wait<S - 1>();
    Raw v[NV];
    uint32_t m = 0;
    unrolled<NV>([&](auto i) {
      if (i * 32 < left) {
        v[i] = load_raw<E, i * kChunk>(ring + stage * kStage);
        m = max(m, amax8_raw<E>(v[i]));
      }
    });
    if (++stage == S) stage = 0;
    m = team_max(__reduce_max_sync(0xffffffffu, m), slots[par], tm, warp);
    const rows8::RowScale q = rows8::row_scale(m);
    if (wt == 0 && lane == 0) scales[r] = q.scale;
    unrolled<NV>([&](auto i) {
      if (i * 32 < left) {
        float f[8];
        Elem<E>::widen(v[i], f);
        rows8::store_codes8(dst + i * 256, f, q.inv);
      }
    });
    dst += step * stride;
  }
}

// Restoring: a group of lanes (a power of two, up to 32) takes `per` chunks of eight
// codes of one row, up to kRestoreChunks per lane, all of them in flight at a time:
// narrow rows share a warp and wide ones are cut into equal segments.
constexpr int kRestoreChunks = 4;  // (of 8: 65536 x 1023 101 us, where 4 then took 70)
struct Restore {
  int group, segments, per;
  int64_t units;
};
__device__ __forceinline__ int64_t row_of(int64_t u, const Restore &p) {
  return p.units <= 0xffffffffll ? int64_t(uint32_t(u) / uint32_t(p.segments)) : u / p.segments;
}

template <class E>
__global__ void __launch_bounds__(kThreads)
row_dequantize_kernel(const int8_t *__restrict__ codes, int64_t stride, const float *__restrict__ scales,
                      E *__restrict__ x, int64_t rows, int C, const Restore p) {
  pdl_wait();
  const int lane = threadIdx.x & (p.group - 1);
  const int64_t hop = (int64_t(gridDim.x) * kThreads) / p.group;
  for (int64_t u = (int64_t(blockIdx.x) * kThreads + threadIdx.x) / p.group; u < p.units; u += hop) {
    const int64_t r = row_of(u, p);
    const int c0 = int(u - r * p.segments) * p.per, end = min(c0 + p.per, C / 8);
    const uint2 *from = reinterpret_cast<const uint2 *>(codes + r * stride);
    const float s = __ldg(scales + r);
    uint2 v[kRestoreChunks];
#pragma unroll
    for (int i = 0; i < kRestoreChunks; ++i)
      if (c0 + lane + i * p.group < end) v[i] = __ldcs(from + c0 + lane + i * p.group);
#pragma unroll
    for (int i = 0; i < kRestoreChunks; ++i) {
      const int c = c0 + lane + i * p.group;
      if (c < end) {
        float f[8];
        restore<kInt8>(v[i], s, f);
        st8(x + r * C + int64_t(c) * 8, f);
      }
    }
  }
}

// The same for rows of any width: the chunks are the aligned ones of x (see
// rows_general.cu), whose codes start anywhere in a word and lie in up to three.
template <class E>
__global__ void __launch_bounds__(kThreads)
row_dequantize_general_kernel(const int8_t *__restrict__ codes, int64_t stride, const float *__restrict__ scales,
                              E *__restrict__ x, int64_t rows, int C, const Restore p) {
  pdl_wait();
  const int lane = threadIdx.x & (p.group - 1);
  const int64_t hop = (int64_t(gridDim.x) * kThreads) / p.group;
  for (int64_t u = (int64_t(blockIdx.x) * kThreads + threadIdx.x) / p.group; u < p.units; u += hop) {
    const int64_t r = row_of(u, p);
    const int a = int((r * C) & 7), c0 = int(u - r * p.segments) * p.per, end = min(c0 + p.per, (a + C + 7) >> 3);
    const int8_t *row = codes + r * stride;
    const float s = __ldg(scales + r);
    const auto whole = [&](int at) { return __ldg(reinterpret_cast<const uint32_t *>(row + at)); };
    const auto single = [&](int at) { return __ldg(row + at); };
    uint2 v[kRestoreChunks];
#pragma unroll
    for (int i = 0; i < kRestoreChunks; ++i) {
      const int c = c0 + lane + i * p.group, e = 8 * c - a;
      if (c < end) {
        uint32_t q[3];
        code_words(e & ~3, C, whole, single, q);
        v[i] = make_uint2(__funnelshift_r(q[0], q[1], 8 * (e & 3)), __funnelshift_r(q[1], q[2], 8 * (e & 3)));
      }
    }
#pragma unroll
    for (int i = 0; i < kRestoreChunks; ++i) {
      const int c = c0 + lane + i * p.group, e = 8 * c - a;
      if (c < end) {
        float f[8];
        restore<kInt8>(v[i], s, f);
        E *to = x + r * C + e;
        if (e >= 0 && e + 8 <= C) {
          st8(to, f);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (e + k >= 0 && e + k < C) to[k] = Elem<E>::narrow1(f[k]);
        }
      }
    }
  }
}

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
                         int64_t rows, int C, bool vec, cudaStream_t s) {
  FMHC_DISPATCH_ELEM(dtype, {
    Shape p;
    if (vec && (C % 8 != 0 || C <= 128)) {
      if (launch_general_fwd(x, dtype, nullptr, nullptr, 0, 0.f, nullptr, nullptr, nullptr, codes, stride, scales, false,
                             rows, C, s))
        return;
    } else if (vec && register_shape(rows, C, kMaxNV<E>, kQuantWarps, &p)) {
      auto k = p.nv == 1 ? row_quantize_kernel<E, 1> : p.nv == 2 ? row_quantize_kernel<E, 2> : row_quantize_kernel<E, kMaxNV<E>>;
      const size_t smem = size_t(p.threads) * kStages<E> * p.nv * sizeof(typename Elem<E>::Raw);
      allow_smem(reinterpret_cast<const void *>(k), smem);
      launch(k, dim3(blocks_for(rows, p)), dim3(p.threads), smem, s, (const E *)x, (int8_t *)codes, stride, scales,
             rows, C, p.team);
      return;
    }
    auto k = row_quantize_any_kernel<E>;
    launch(k, dim3(grid_for(k, rows * kWarps, kThreads)), dim3(kThreads), 0, s, (const E *)x,
           (int8_t *)codes, stride, scales, rows, C);
  });
}

void launch_row_dequantize(const void *codes, int64_t stride, const float *scales, void *x, int dtype,
                           int64_t rows, int C, bool vec, cudaStream_t s) {
  FMHC_DISPATCH_ELEM(dtype, {
    if (vec) {
      const int chunks = C % 8 ? (C + 14) / 8 : C / 8;  // of a row, wherever it starts
      Restore p{1, 0, 0, 0};
      while (p.group < 32 && p.group < chunks) p.group *= 2;
      p.segments = (chunks + kRestoreChunks * p.group - 1) / (kRestoreChunks * p.group);
      p.per = (chunks + p.segments - 1) / p.segments;
      p.units = rows * p.segments;
      auto k = C % 8 ? row_dequantize_general_kernel<E> : row_dequantize_kernel<E>;
      launch(k, dim3(grid_for(k, (p.units * p.group + 31) / 32, kThreads)), dim3(kThreads), 0, s, (const int8_t *)codes,
             stride, scales, (E *)x, rows, C, p);
      return;
    }
    auto k = row_dequantize_any_kernel<E>;
    launch(k, dim3(grid_for(k, rows * kWarps, kThreads)), dim3(kThreads), 0, s, (const int8_t *)codes,
           stride, scales, (E *)x, rows, C);
  });
}

}  // namespace fmhc
