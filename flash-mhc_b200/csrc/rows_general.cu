// Root-mean-square norm, and putting rows into 8 bits, for rows of any width: those
// that start anywhere in a 16-byte word (C % 8 != 0), and those of fewer than 17 chunks
// of eight values, which share a warp.  (rms_norm.cu and rows8.cu have the kernels for
// wide rows of whole chunks, and for pointers that are not 16-byte aligned.)
//
// Chunks are the aligned ones of memory: chunk j of a row holds its values
// 8 j - a .. 8 j - a + 7, a being where the row starts in its first chunk, so that
// loads and most stores are whole words; what a row's first and last chunk hold of its
// neighbours is masked.  A lane's rows are a multiple of 8 / gcd(C, 8) apart and so
// start at the same a: a lane has the same columns in every row, with the weight and
// the weight's gradient in registers.  Narrow rows take a power-of-two group of lanes
// each, 32 / group of them in a warp.
//
// Measured, bf16, us: one block per row (rms_norm.cu, rows8.cu) / these (the bytes at the
// copy rate).
//                       131072 x 64          131072 x 77          65536 x 1023
//   norm                20 / 10.5 (5.2)      168 / 19 (6.2)       162 / 72 (41)
//   backward            33 / 17 (7.7)        196 / 32 (9.3)       430 / 121 (62)
//   add, norm, 8 bits   35 / 16 (9.0)        256 / 39 (11)        317 / 159 (72)
//   quantise            21 / 10.5 (3.9)      120 / 25 (4.7)       107 / 97 (31)
// (64: the kernels for wide rows, a warp per row, in place of a block.)  Instructions
// bound them (70 % of the issue slots at 1023): masks, the ends' stores value by value,
// and codes moved between lanes.
#include "rows_general.h"

#include <numeric>

#include "fmhc_launch.h"
#include "norm_rows.cuh"
#include "rows8.cuh"

namespace fmhc {

using namespace act8;
using namespace norm_rows;

namespace {

constexpr int kFwdWarps = 24;  // per block, one block per SM
constexpr int kBwdWarps = 16;
constexpr int kMaxNV = 2;      // chunks per lane: the weight's columns take 8 registers each
constexpr int kStages = 2;     // rows in flight in the ring

// What a lane holds of its rows.
struct Part {
  int a;     // where the row starts in its first chunk
  int c0;    // first chunk; the next is 32 on
  int left;  // chunk i exists if i * 32 < left
  int C;
  __device__ __forceinline__ Part(int64_t row, int C_, int first) : a(int((row * C_) & 7)), c0(first), C(C_) {
    left = ((a + C + 7) >> 3) - c0;
  }
  __device__ __forceinline__ int element(int i) const { return 8 * (c0 + 32 * i) - a; }  // of the chunk's first value
  __device__ __forceinline__ int lo(int i) const { return max(-element(i), 0); }
  __device__ __forceinline__ int hi(int i) const { return min(C - element(i), 8); }
  __device__ __forceinline__ bool whole(int i) const { return element(i) >= 0 && element(i) + 8 <= C; }
};

__device__ __forceinline__ void mask8(float (&f)[8], const Part &p, int i) {
  if (p.whole(i)) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = k >= p.lo(i) && k < p.hi(i) ? f[k] : 0.f;
}
template <class E>
__device__ __forceinline__ void store_part(E *to, const float (&f)[8], const Part &p, int i) {
  if (p.whole(i)) {
    st8(to, f);
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k >= p.lo(i) && k < p.hi(i)) to[k] = Elem<E>::narrow1(f[k]);
}

// A chunk into shared memory, of which `there` values lie before the tensor's end.
__device__ __forceinline__ void copy16_upto(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
template <class E, int OFF>
__device__ __forceinline__ void copy_part(uint32_t dst, const E *src, int64_t there) {
  if (there >= 8) {
    copy_raw<E, OFF>(dst, src);
  } else {
    const int bytes = int(there) * int(sizeof(E));
    copy16_upto(dst + OFF, src, min(bytes, 16));
    if constexpr (sizeof(E) == 4) copy16_upto(dst + OFF + 16, bytes > 16 ? src + 4 : src, max(bytes - 16, 0));
  }
}

__device__ __forceinline__ uint32_t group_most(uint32_t v, int group) {
  for (int o = group >> 1; o >= 1; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Weight's columns of a lane; 0 where it holds none.
template <int NV>
__device__ __forceinline__ void load_weight(const void *w, int pdt, const Part &p, float (&fw)[NV][8]) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = p.element(i) + k;
      fw[i][k] = i * 32 < p.left && c >= 0 && c < p.C ? param1(w, pdt, c, 1.f) : 0.f;
    }
}

__device__ __forceinline__ void store_bytes(int8_t *to, uint2 v, int n) {
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < n) to[k] = int8_t((k < 4 ? v.x : v.y) >> (8 * (k & 3)));
}
// The codes of a row start at a multiple of 8 bytes, its chunks a bytes further: block
// j of eight codes is the end of chunk j and the beginning of chunk j + 1, which
// the next lane has.
template <int NV>
__device__ __forceinline__ void store_codes(int8_t *row, const uint2 (&q)[NV], const Part &p, bool valid, int lane,
                                            int group, bool first_warp) {
  const int gl = lane & (group - 1), next = (lane & ~(group - 1)) | ((gl + 1) & (group - 1));
  const bool near = p.a < 4;  // the block starts in the chunk's first word
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint2 own = q[i], send = i + 1 < NV && gl == 0 && group == 32 ? q[i + 1 < NV ? i + 1 : i] : own;
    const uint32_t x = __shfl_sync(0xffffffffu, send.x, next), y = __shfl_sync(0xffffffffu, send.y, next);
    // Not in this warp: the chunk after the last one of a warp that is not the row's last.
    const bool beyond = p.a != 0 && group == 32 && lane == 31 && i + 1 == NV && i * 32 + 1 < p.left;
    if (valid && i * 32 < p.left) {
      const int block = 8 * (p.c0 + 32 * i);  // first element
      const uint32_t w0 = near ? own.x : own.y, w1 = near ? own.y : x, w2 = near ? x : y;
      const uint2 v = make_uint2(__funnelshift_r(w0, w1, 8 * p.a), __funnelshift_r(w1, w2, 8 * p.a));
      const int n = min(beyond ? 8 - p.a : 8, p.C - block);
      if (n == 8) __stcs(reinterpret_cast<uint2 *>(row + block), v);
      else store_bytes(row + block, v, n);
      // What the warp before has not.
      if (i == 0 && lane == 0 && !first_warp) store_bytes(row + p.element(0), own, min(p.a, p.C - p.element(0)));
    }
  }
}

// -------------------------------------------------------------------- forward
// RES: with a residual.  CODES: the output as codes and scales.  NORM false: x itself
// is put into 8 bits.
template <class E, int NV, bool RES, bool CODES, bool NORM>
__global__ void __launch_bounds__(32 * kFwdWarps, 1)
general_fwd_kernel(const E *__restrict__ x, const E *__restrict__ res, const void *__restrict__ w, int pdt,
                   float eps, E *__restrict__ y, E *__restrict__ total, float *__restrict__ rstd_out,
                   int8_t *__restrict__ codes, int64_t stride, float *__restrict__ scales, int64_t rows, int C,
                   int team, int group) {
  using Raw = typename Elem<E>::Raw;
  constexpr int S = kStages;
  constexpr int kChunk = 32 * int(sizeof(Raw)), kStage = NV * kChunk * (RES ? 2 : 1);
  extern __shared__ uint4 dyn[];
  __shared__ float sum_slots[2][kFwdWarps];
  __shared__ uint32_t max_slots[2][kFwdWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int teams = (blockDim.x >> 5) / team, wt = warp % team;
  const Team tm(team, warp, lane);
  const int per_warp = 32 / group, sub = lane / group;
  const uint32_t ring = shared_addr(dyn) + warp * (S * kStage) + lane * int(sizeof(Raw));
  const int64_t step = int64_t(gridDim.x) * teams * per_warp;
  int64_t base = (int64_t(blockIdx.x) * teams + warp / team) * per_warp;  // the warp's first row
  const Part p(base + sub, C, wt * NV * 32 + (lane & (group - 1)));
  const float inv_C = 1.f / float(C);
  pdl_wait();
  const int64_t end = rows * C;
  int64_t at = (base + sub) * C + p.element(0);  // of the lane's first chunk, in the tensors
  int64_t fetched = base + sub, from_at = at;
  const auto fetch = [&](int stage) {
    if (fetched < rows) {
      unrolled<NV>([&](auto i) {
        if (i * 32 < p.left) {
          const int64_t c = from_at + i * 256;
          copy_part<E, i * kChunk>(ring + stage * kStage, x + c, end - c);
          if constexpr (RES) copy_part<E, (NV + i) * kChunk>(ring + stage * kStage, res + c, end - c);
        }
      });
    }
    fetched += step;
    from_at += step * C;
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s);
  float fw[NV][8];
  if constexpr (NORM) load_weight(w, pdt, p, fw);
  int par = 0, stage = 0;
  for (; base < rows; base += step, at += step * C, par ^= 1) {
    fetch(stage == 0 ? S - 1 : stage - 1);
    copy_wait<S - 1>();
    const int64_t r = base + sub;
    const bool valid = r < rows;
    float f[NV][8];
    float q = 0.f;
    unrolled<NV>([&](auto i) {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[i][k] = 0.f;
      if (valid && i * 32 < p.left) {
        Elem<E>::widen(load_raw<E, i * kChunk>(ring + stage * kStage), f[i]);
        if constexpr (RES) {
          float g[8];
          Elem<E>::widen(load_raw<E, (NV + i) * kChunk>(ring + stage * kStage), g);
#pragma unroll
          for (int k = 0; k < 8; ++k) f[i][k] += g[k];
          Elem<E>::widen(Elem<E>::narrow(f[i]), f[i]);
          store_part(total + at + i * 256, f[i], p, i);
        }
        mask8(f[i], p, i);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) q = fmaf(f[i][k], f[i][k], q);
    });
    if (++stage == S) stage = 0;
    if constexpr (NORM) {
      q = team_sum1(group_sum(q, group), sum_slots[par], tm, warp);
      const float rstd = rsqrtf(fmaf(q, inv_C, eps));
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) f[i][k] = f[i][k] * rstd * fw[i][k];
      // A column that this lane has not is 0 times a weight of 0, but not under an
      // infinite or NaN rstd.
      if constexpr (CODES) unrolled<NV>([&](auto i) { mask8(f[i], p, i); });
      if constexpr (!CODES) {
        if (valid && (lane & (group - 1)) == 0 && wt == 0) rstd_out[r] = rstd;
        unrolled<NV>([&](auto i) {
          if (valid && i * 32 < p.left) store_part(y + at + i * 256, f[i], p, i);
        });
      }
    }
    if constexpr (CODES) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i * 32 < p.left) {
#pragma unroll
          for (int k = 0; k < 8; ++k) m = max(m, rows8::magnitude(f[i][k]));
        }
      m = team_max(group_most(m, group), max_slots[par], tm, warp);
      const rows8::RowScale sc = rows8::row_scale(m);
      if (valid && (lane & (group - 1)) == 0 && wt == 0) scales[r] = sc.scale;
      uint2 out[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i)
        out[i] = make_uint2(rows8::code4(f[i][0], f[i][1], f[i][2], f[i][3], sc.inv),
                            rows8::code4(f[i][4], f[i][5], f[i][6], f[i][7], sc.inv));
      store_codes<NV>(codes + r * stride, out, p, valid, lane, group, wt == 0);
    }
  }
}

// ------------------------------------------------------------------- backward
template <class E, int NV, bool THIRD>
__global__ void __launch_bounds__(32 * kBwdWarps, 1)
general_bwd_kernel(const E *__restrict__ g, const E *__restrict__ gt, const E *__restrict__ x,
                   const float *__restrict__ rstd, const void *__restrict__ w, int pdt, E *__restrict__ gx,
                   float *__restrict__ part, int64_t rows, int C, int team, int group) {
  using Raw = typename Elem<E>::Raw;
  constexpr int S = kStages;
  constexpr int kChunk = 32 * int(sizeof(Raw)), kStage = NV * kChunk * (THIRD ? 3 : 2);
  constexpr int kRow = 128;  // rstd of up to 32 rows, per warp and stage
  extern __shared__ uint4 dyn[];
  __shared__ float slots[2][kBwdWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int teams = warps / team, wt = warp % team;
  const Team tm(team, warp, lane);
  const int per_warp = 32 / group, sub = lane / group;
  const uint32_t ring = shared_addr(dyn) + warp * (S * kStage) + lane * int(sizeof(Raw));
  // Copied by one lane of a group for all of it: a warp barrier stands on both sides of
  // a refill.
  const uint32_t ring_r = shared_addr(dyn) + warps * (S * kStage) + warp * (S * kRow) + sub * 4;
  const int64_t step = int64_t(gridDim.x) * teams * per_warp;
  int64_t base = (int64_t(blockIdx.x) * teams + warp / team) * per_warp;
  const Part p(base + sub, C, wt * NV * 32 + (lane & (group - 1)));
  const float inv_C = 1.f / float(C);
  pdl_wait();
  const int64_t end = rows * C;
  int64_t at = (base + sub) * C + p.element(0);
  int64_t fetched = base + sub, from_at = at;
  const auto fetch = [&](int stage) {
    if (fetched < rows) {
      if ((lane & (group - 1)) == 0) copy_async4(ring_r + stage * kRow, rstd + fetched);
      unrolled<NV>([&](auto i) {
        if (i * 32 < p.left) {
          const int64_t c = from_at + i * 256;
          copy_part<E, i * kChunk>(ring + stage * kStage, g + c, end - c);
          copy_part<E, (NV + i) * kChunk>(ring + stage * kStage, x + c, end - c);
          if constexpr (THIRD) copy_part<E, (2 * NV + i) * kChunk>(ring + stage * kStage, gt + c, end - c);
        }
      });
    }
    fetched += step;
    from_at += step * C;
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s);
  float fw[NV][8], dw[NV][8];
  load_weight(w, pdt, p, fw);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) dw[i][k] = 0.f;
  int par = 0, stage = 0;
  for (; base < rows; base += step, at += step * C, par ^= 1) {
    __syncwarp();
    fetch(stage == 0 ? S - 1 : stage - 1);
    copy_wait<S - 1>();
    __syncwarp();
    const bool valid = base + sub < rows;
    const float rs = valid ? load_shared_f32(ring_r + stage * kRow) : 0.f;
    const uint32_t from = ring + stage * kStage;
    float fg[NV][8], fx[NV][8];
    float dot = 0.f;
    unrolled<NV>([&](auto i) {
#pragma unroll
      for (int k = 0; k < 8; ++k) fg[i][k] = fx[i][k] = 0.f;
      if (valid && i * 32 < p.left) {
        Elem<E>::widen(load_raw<E, i * kChunk>(from), fg[i]);
        Elem<E>::widen(load_raw<E, (NV + i) * kChunk>(from), fx[i]);
        mask8(fg[i], p, i);
        mask8(fx[i], p, i);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float gxh = fg[i][k] * (fx[i][k] * rs);
          dw[i][k] += gxh;
          dot = fmaf(gxh, fw[i][k], dot);
        }
      }
    });
    const float sum = team_sum1(group_sum(dot, group), slots[par], tm, warp);
    const float c = -sum * inv_C * rs;  // times x
    unrolled<NV>([&](auto i) {
      if (valid && i * 32 < p.left) {
        float ft[8], o[8];
        if constexpr (THIRD) Elem<E>::widen(load_raw<E, (2 * NV + i) * kChunk>(from), ft);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float v = fmaf(fx[i][k], c, fg[i][k] * fw[i][k]);
          o[k] = THIRD ? fmaf(rs, v, ft[k]) : rs * v;
        }
        store_part(gx + at + i * 256, o, p, i);
      }
    });
    if (++stage == S) stage = 0;
  }
  if (part == nullptr) return;
  // Join the block's rows in the ring's memory (no copy is in flight), in their order.
  copy_wait<0>();
  __syncthreads();
  float *sums = reinterpret_cast<float *>(dyn);  // [teams * per_warp][C]
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * 32 < p.left) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k >= p.lo(i) && k < p.hi(i)) sums[(warp / team * per_warp + sub) * C + p.element(i) + k] = dw[i][k];
    }
  __syncthreads();
  float *out = part + int64_t(blockIdx.x) * C;
  for (int c1 = threadIdx.x; c1 < C; c1 += blockDim.x) {
    float v = 0.f;
    for (int t = 0; t < teams * per_warp; ++t) v += sums[t * C + c1];
    out[c1] = v;
  }
}

// ------------------------------------------------------------------ launchers
struct Split {
  int team, nv, teams, group, grid;
  int threads() const { return teams * team * 32; }
};
// Rows over groups, warps and teams; false for rows that are too wide.
bool split_for(int64_t rows, int C, int max_warps, Split *p) {
  const int chunks = C % 8 ? (C + 14) / 8 : C / 8;  // of a row, wherever it starts
  if (chunks > 32 * kMaxNV * kMaxTeam) return false;
  p->team = p->nv = 1;
  p->group = 32;
  if (chunks <= 16) {
    while (p->group / 2 >= chunks) p->group /= 2;
  } else {
    if (chunks > 32) p->nv = kMaxNV;
    p->team = (chunks + 32 * p->nv - 1) / (32 * p->nv);
  }
  const int sms = sm_count(), per_warp = 32 / p->group;
  const int64_t want = (rows + int64_t(sms) * per_warp - 1) / (int64_t(sms) * per_warp);
  p->teams = int(std::min<int64_t>(std::max<int64_t>(want, 1), max_warps / p->team));
  const int64_t per_block = int64_t(p->teams) * per_warp;
  p->grid = int(std::min<int64_t>((rows + per_block - 1) / per_block, sms));
  // Rows that a lane takes one after another have to start at the same place in a chunk.
  const int period = 8 / std::gcd(C, 8);
  if (rows > p->grid * per_block)
    while (p->grid > 1 && (p->grid * per_block) % period) --p->grid;
  return p->grid * per_block % period == 0 || rows <= p->grid * per_block;
}

#define FMHC_DISPATCH_NV(NV_RT, ...)                         \
  do {                                                       \
    if ((NV_RT) == 1) { constexpr int NV = 1; __VA_ARGS__; } \
    else { constexpr int NV = kMaxNV; __VA_ARGS__; }         \
  } while (0)

template <class E, bool RES, bool CODES, bool NORM>
void launch_fwd(const Split &p, const void *x, const void *res, const void *w, int pdt, float eps, void *y,
                void *total, float *rstd, void *codes, int64_t stride, float *scales, int64_t rows, int C,
                cudaStream_t s) {
  FMHC_DISPATCH_NV(p.nv, {
    auto k = general_fwd_kernel<E, NV, RES, CODES, NORM>;
    const size_t smem = size_t(p.threads()) * kStages * NV * sizeof(typename Elem<E>::Raw) * (RES ? 2 : 1);
    allow_smem(reinterpret_cast<const void *>(k), smem);
    launch(k, dim3(p.grid), dim3(p.threads()), smem, s, (const E *)x, (const E *)res, w, pdt, eps, (E *)y, (E *)total,
           rstd, (int8_t *)codes, stride, scales, rows, C, p.team, p.group);
  });
}

}  // namespace

bool launch_general_fwd(const void *x, int dtype, const void *res, const void *w, int pdt, float eps, void *y,
                        void *total, float *rstd, void *codes, int64_t stride, float *scales, bool norm,
                        int64_t rows, int C, cudaStream_t s) {
  Split p;
  if (!split_for(rows, C, kFwdWarps, &p)) return false;
  FMHC_DISPATCH_ELEM(dtype, {
    auto k = !norm ? launch_fwd<E, false, true, false>
           : res != nullptr ? codes != nullptr ? launch_fwd<E, true, true, true> : launch_fwd<E, true, false, true>
                            : codes != nullptr ? launch_fwd<E, false, true, true> : launch_fwd<E, false, false, true>;
    k(p, x, res, w, pdt, eps, y, total, rstd, codes, stride, scales, rows, C, s);
  });
  return true;
}

int general_bwd_parts(int64_t rows, int C) {
  Split p;
  return split_for(rows, C, kBwdWarps, &p) ? p.grid : 0;
}

bool launch_general_bwd(const void *g, int dtype, const void *gt, const void *x, const float *rstd, const void *w,
                        int pdt, void *gx, float *part, int64_t rows, int C, cudaStream_t s) {
  Split p;
  if (!split_for(rows, C, kBwdWarps, &p)) return false;
  FMHC_DISPATCH_ELEM(dtype, FMHC_DISPATCH_NV(p.nv, {
    const bool third = gt != nullptr;
    auto k = third ? general_bwd_kernel<E, NV, true> : general_bwd_kernel<E, NV, false>;
    const size_t smem = size_t(p.threads()) * kStages * NV * sizeof(typename Elem<E>::Raw) * (third ? 3 : 2) +
                        size_t(p.threads() / 32) * kStages * 128;
    allow_smem(reinterpret_cast<const void *>(k), smem);
    launch(k, dim3(p.grid), dim3(p.threads()), smem, s, (const E *)g, (const E *)gt, (const E *)x, rstd, w, pdt,
           (E *)gx, part, rows, C, p.team, p.group);
  }));
  return true;
}

}  // namespace fmhc
