// Layer norm over rows of C values, forward and backward, with the input kept
// as it is or in 8 bits (act8.cuh).
//
//   mean = <x>, rstd = 1 / sqrt(<(x - mean)^2> + eps)      (<> : mean over C)
//   y    = (x - mean) rstd w + b
//   grad_x = rstd (gw - <gw> - xh <gw xh>),  gw = g w,  xh = (x - mean) rstd
//   grad_w = sum over rows of g xh,  grad_b = sum over rows of g
//
// The backward from a checkpoint puts the restored x in xh and keeps mean and
// rstd, which are those of the true x.
//
// Statistics, sums and gradients are f32.  The variance is taken about the
// mean, never as <x^2> - mean^2: each warp sums the squares about its own mean
// and warps are joined by  M2 = sum M2_w + n_w (mean_w - mean)^2.
//
// One pass over the data: a team of 1..8 warps holds a row in registers (NV
// chunks of eight values per lane), so x is read once forward, and x and g once
// backward.  Backward, a lane keeps the same columns for every row its team
// takes, so its share of grad_w and grad_b stays in registers until the end;
// blocks write one partial each, and a small kernel adds the partials in block
// order (no atomics: the same bits every time).
#include "act8.cuh"
#include "fmhc_launch.h"
#include "grid.cuh"

#include <algorithm>

namespace fmhc {

using namespace act8;

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTeam = kWarps;  // warps per row
constexpr int kMaxNV = 4;         // chunks of eight values per lane
constexpr int kMaxParts = 1024;

// w or b at column c, in the parameters' own type (fmhc_dtype); `def` if absent.
__device__ __forceinline__ float param1(const void *p, int dtype, int64_t c, float def) {
  if (p == nullptr) return def;
  if (dtype == 0) return __ldg(reinterpret_cast<const float *>(p) + c);
  if (dtype == 1) return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[c]);
  return __half2float(reinterpret_cast<const __half *>(p)[c]);
}
__device__ __forceinline__ void param8(const void *p, int dtype, int c, float def, float (&f)[8]) {
  if (p == nullptr) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = def;
  } else if (dtype == 0) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p) + c * 2);
    const float4 b = __ldg(reinterpret_cast<const float4 *>(p) + c * 2 + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const uint4 r = __ldg(reinterpret_cast<const uint4 *>(p) + c);
    if (dtype == 1) Elem<__nv_bfloat16>::widen(r, f);
    else Elem<__half>::widen(r, f);
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Adds a pair over the `team` warps of a row.  `slot` holds one float2 per warp
// of the block, one array for even and one for odd rows of a team, so one
// barrier per row is enough: a warp writes a slot again two rows later, after
// the barrier of the row between, which no warp reaches before it has read.
// Each team has a named barrier of its own (1 + team index), since teams take
// different numbers of rows.
__device__ __forceinline__ float2 team_sum(float2 v, float2 *slot, int team, int warp, int lane) {
  if (team == 1) return v;
  const int first = warp / team * team;
  if (lane == 0) slot[warp] = v;
  named_bar_sync(1 + warp / team, team * 32);
  float2 t = slot[first];
  for (int i = 1; i < team; ++i) {
    const float2 o = slot[first + i];
    t.x += o.x;
    t.y += o.y;
  }
  return t;
}

// -------------------------------------------------------------------- forward
template <class E, int NV, int FMT>
__global__ void __launch_bounds__(kThreads)
ln_fwd_kernel(const E *__restrict__ x, const void *__restrict__ w, const void *__restrict__ b,
              int pdt, float eps, E *__restrict__ y, float *__restrict__ mean_out,
              float *__restrict__ rstd_out, uint8_t *__restrict__ codes,
              uint8_t *__restrict__ scales, int64_t rows, int C, int team) {
  __shared__ float2 slots[2][kWarps];
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int teams = kWarps / team;
  const int wt = warp % team;
  const int nchunk = C / 8, nb = (C + kBlock - 1) / kBlock;
  // Values of this warp: chunks wt * 32 + lane + i * 32 * team below nchunk.
  int mine = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) mine += min(max(nchunk - (wt + i * team) * 32, 0), 32) * 8;
  const float inv_mine = mine ? 1.f / float(mine) : 0.f, inv_C = 1.f / float(C);
  int par = 0;
  for (int64_t r = int64_t(blockIdx.x) * teams + warp / team; r < rows;
       r += int64_t(gridDim.x) * teams, par ^= 1) {
    float f[NV][8];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (wt + i * team) * 32 + lane;
      typename Elem<E>::Raw raw = {};
      if (c < nchunk) raw = ld8(x + r * C + c * 8);
      Elem<E>::widen(raw, f[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) s += f[i][k];
    s = warp_sum(s);
    const float m_w = s * inv_mine;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((wt + i * team) * 32 + lane < nchunk) {
#pragma unroll
        for (int k = 0; k < 8; ++k) q = fmaf(f[i][k] - m_w, f[i][k] - m_w, q);
      }
    q = warp_sum(q);
    float mean = m_w, m2 = q;
    if (team > 1) {
      // Join the warps: means first, then the squares about the row's mean.
      const int first = warp / team * team;
      float2 *slot = slots[par];
      if (lane == 0) slot[warp] = make_float2(s, q);
      named_bar_sync(1 + warp / team, team * 32);
      float total = 0.f;
      for (int i = 0; i < team; ++i) total += slot[first + i].x;
      mean = total * inv_C;
      m2 = 0.f;
      for (int i = 0; i < team; ++i) {
        int n = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) n += min(max(nchunk - (i + v * team) * 32, 0), 32) * 8;
        if (n) {
          const float2 o = slot[first + i];
          const float d = o.x / float(n) - mean;
          m2 += fmaf(float(n) * d, d, o.y);
        }
      }
    }
    const float rstd = rsqrtf(fmaf(m2, inv_C, eps));
    if (wt == 0 && lane == 0) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (wt + i * team) * 32 + lane;
      uint32_t e = 0;
      if constexpr (FMT != kNone) e = scale_byte<FMT>(amax_block(amax8(f[i])));
      if (c < nchunk) {
        if constexpr (FMT != kNone) {
          __stcs(reinterpret_cast<uint2 *>(codes + r * C + c * 8), encode8<FMT>(f[i], e));
          if ((lane & 3) == 0) __stcs(scales + r * nb + (c >> 2), uint8_t(e));
        }
        float fw[8], fb[8], o[8];
        param8(w, pdt, c, 1.f, fw);
        param8(b, pdt, c, 0.f, fb);
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = fmaf((f[i][k] - mean) * rstd, fw[k], fb[k]);
        st8(y + r * C + c * 8, o);
      }
    }
  }
}

// ------------------------------------------------------------------- backward
template <class E, int NV, int FMT>
__global__ void __launch_bounds__(kThreads)
ln_bwd_kernel(const E *__restrict__ g, const void *__restrict__ x,
              const uint8_t *__restrict__ scales, const float *__restrict__ mean,
              const float *__restrict__ rstd, const void *__restrict__ w, int pdt,
              E *__restrict__ gx, float *__restrict__ part, int64_t rows, int C, int team) {
  __shared__ float2 slots[2][kWarps];
  extern __shared__ float joined[];  // [2][C], when a block has several teams
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int teams = kWarps / team;
  const int wt = warp % team;
  const int nchunk = C / 8, nb = (C + kBlock - 1) / kBlock;
  const float inv_C = 1.f / float(C);
  float dw[NV][8], db[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) dw[i][k] = db[i][k] = 0.f;
  int par = 0;
  for (int64_t r = int64_t(blockIdx.x) * teams + warp / team; r < rows;
       r += int64_t(gridDim.x) * teams, par ^= 1) {
    const float m = __ldg(mean + r), rs = __ldg(rstd + r);
    float xh[NV][8], gw[NV][8];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (wt + i * team) * 32 + lane;
#pragma unroll
      for (int k = 0; k < 8; ++k) xh[i][k] = gw[i][k] = 0.f;
      if (c < nchunk) {
        float fg[8], fw[8];
        if constexpr (FMT == kNone) {
          Elem<E>::widen(ld8(reinterpret_cast<const E *>(x) + r * C + c * 8), xh[i]);
        } else {
          const Codes<8> q = ld_codes<8>(reinterpret_cast<const uint8_t *>(x) + r * C + c * 8);
          restore<FMT, 8>(q, scale_value(__ldg(scales + r * nb + (c >> 2))), xh[i]);
        }
        Elem<E>::widen(ld8(g + r * C + c * 8), fg);
        param8(w, pdt, c, 1.f, fw);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          xh[i][k] = (xh[i][k] - m) * rs;
          gw[i][k] = fg[k] * fw[k];
          dw[i][k] = fmaf(fg[k], xh[i][k], dw[i][k]);
          db[i][k] += fg[k];
          s.x += gw[i][k];
          s.y = fmaf(gw[i][k], xh[i][k], s.y);
        }
      }
    }
    s.x = warp_sum(s.x);
    s.y = warp_sum(s.y);
    s = team_sum(s, slots[par], team, warp, lane);
    const float c1 = s.x * inv_C, c2 = s.y * inv_C;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (wt + i * team) * 32 + lane;
      if (c < nchunk) {
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = rs * (gw[i][k] - fmaf(xh[i][k], c2, c1));
        st8(gx + r * C + c * 8, o);
      }
    }
  }
  if (part == nullptr) return;
  // Join the block's teams in team order, then write the block's partial.
  float *dst = part + int64_t(blockIdx.x) * 2 * C;
  for (int t = 0; t < teams; ++t) {
    if (warp / team == t) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (wt + i * team) * 32 + lane;
        if (c < nchunk) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float a = dw[i][k], d = db[i][k];
            if (t > 0) {
              a += joined[c * 8 + k];
              d += joined[C + c * 8 + k];
            }
            if (t == teams - 1) {
              dst[c * 8 + k] = a;
              dst[C + c * 8 + k] = d;
            } else {
              joined[c * 8 + k] = a;
              joined[C + c * 8 + k] = d;
            }
          }
        }
      }
    }
    if (t < teams - 1) __syncthreads();
  }
}

// Adds the partials [n][2][C] in order: grad_w and grad_b in the parameters'
// type.  Either may be absent.  A block takes 32 columns; each of its 8 warps
// adds every eighth partial, and the eight sums are added in warp order.
__global__ void __launch_bounds__(256)
ln_param_grad_kernel(const float *__restrict__ part, void *__restrict__ gw, void *__restrict__ gb,
                     int pdt, int n, int C) {
  pdl_wait();
  __shared__ float acc[2][8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float a = 0.f, d = 0.f;
  if (c < C) {
    for (int i = warp; i < n; i += 8) {
      a += part[int64_t(i) * 2 * C + c];
      d += part[int64_t(i) * 2 * C + C + c];
    }
  }
  acc[0][warp][lane] = a;
  acc[1][warp][lane] = d;
  __syncthreads();
  if (warp < 2 && c < C) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += acc[warp][i][lane];
    void *dst = warp == 0 ? gw : gb;
    if (dst != nullptr) {
      if (pdt == 0) reinterpret_cast<float *>(dst)[c] = s;
      else if (pdt == 1) reinterpret_cast<__nv_bfloat16 *>(dst)[c] = __float2bfloat16_rn(s);
      else reinterpret_cast<__half *>(dst)[c] = __float2half_rn(s);
    }
  }
}

// ---------------------------------------------- any width and any alignment
// One block per row; the row is read again for each step (from L1 or L2).
__device__ float2 block_sum(float2 v, float2 *sh) {
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  __syncthreads();  // the previous use of sh is over
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float2 t = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    t.x += sh[i].x;
    t.y += sh[i].y;
  }
  return t;
}

template <class E, int FMT>
__global__ void __launch_bounds__(kThreads)
ln_fwd_any_kernel(const E *__restrict__ x, const void *__restrict__ w, const void *__restrict__ b,
                  int pdt, float eps, E *__restrict__ y, float *__restrict__ mean_out,
                  float *__restrict__ rstd_out, uint8_t *__restrict__ codes,
                  uint8_t *__restrict__ scales, int64_t rows, int C) {
  __shared__ float2 sh[kWarps];
  pdl_wait();
  const int nb = (C + kBlock - 1) / kBlock, lane = threadIdx.x & 31;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const E *xr = x + r * C;
    float2 v = make_float2(0.f, 0.f);
    for (int c = threadIdx.x; c < C; c += kThreads) v.x += Elem<E>::widen1(xr[c]);
    const float mean = block_sum(v, sh).x / float(C);
    v = make_float2(0.f, 0.f);
    for (int c = threadIdx.x; c < C; c += kThreads) {
      const float d = Elem<E>::widen1(xr[c]) - mean;
      v.x = fmaf(d, d, v.x);
    }
    const float rstd = rsqrtf(block_sum(v, sh).x / float(C) + eps);
    if (threadIdx.x == 0) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
    for (int c = threadIdx.x; c < C; c += kThreads)
      y[r * C + c] = Elem<E>::narrow1(fmaf((Elem<E>::widen1(xr[c]) - mean) * rstd,
                                           param1(w, pdt, c, 1.f), param1(b, pdt, c, 0.f)));
    if constexpr (FMT != kNone) {
      for (int k = threadIdx.x >> 5; k < nb; k += kWarps) {  // a warp per block of 32
        const int c = k * kBlock + lane;
        const float f = c < C ? Elem<E>::widen1(xr[c]) : 0.f;
        const uint32_t e = scale_byte<FMT>(
            __reduce_max_sync(0xffffffffu, __float_as_uint(f) & 0x7fffffffu));
        if (c < C) codes[r * C + c] = uint8_t(encode4<FMT>(f, 0.f, 0.f, 0.f, e));
        if (lane == 0) scales[r * nb + k] = uint8_t(e);
      }
    }
  }
}

// x at (row r, column c), from its own values or from codes.
template <class E, int FMT>
__device__ __forceinline__ float input1(const void *x, const uint8_t *scales, int64_t r, int c,
                                        int C, int nb) {
  if constexpr (FMT == kNone) {
    return Elem<E>::widen1(reinterpret_cast<const E *>(x)[r * C + c]);
  } else {
    return decode1<FMT>(reinterpret_cast<const uint8_t *>(x)[r * C + c]) *
           scale_value(scales[r * nb + c / kBlock]);
  }
}

template <class E, int FMT>
__global__ void __launch_bounds__(kThreads)
ln_bwd_any_kernel(const E *__restrict__ g, const void *__restrict__ x,
                  const uint8_t *__restrict__ scales, const float *__restrict__ mean,
                  const float *__restrict__ rstd, const void *__restrict__ w, int pdt,
                  E *__restrict__ gx, int64_t rows, int C) {
  __shared__ float2 sh[kWarps];
  pdl_wait();
  const int nb = (C + kBlock - 1) / kBlock;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float m = mean[r], rs = rstd[r];
    float2 v = make_float2(0.f, 0.f);
    for (int c = threadIdx.x; c < C; c += kThreads) {
      const float gw = Elem<E>::widen1(g[r * C + c]) * param1(w, pdt, c, 1.f);
      v.x += gw;
      v.y = fmaf(gw, (input1<E, FMT>(x, scales, r, c, C, nb) - m) * rs, v.y);
    }
    v = block_sum(v, sh);
    const float c1 = v.x / float(C), c2 = v.y / float(C);
    for (int c = threadIdx.x; c < C; c += kThreads) {
      const float gw = Elem<E>::widen1(g[r * C + c]) * param1(w, pdt, c, 1.f);
      const float xh = (input1<E, FMT>(x, scales, r, c, C, nb) - m) * rs;
      gx[r * C + c] = Elem<E>::narrow1(rs * (gw - fmaf(xh, c2, c1)));
    }
  }
}

// Partials of grad_w and grad_b: block (cols of 32, slice of rows).
template <class E, int FMT>
__global__ void __launch_bounds__(256)
ln_param_part_any_kernel(const E *__restrict__ g, const void *__restrict__ x,
                         const uint8_t *__restrict__ scales, const float *__restrict__ mean,
                         const float *__restrict__ rstd, float *__restrict__ part, int64_t rows,
                         int C) {
  __shared__ float acc[2][8][32];
  pdl_wait();
  const int nb = (C + kBlock - 1) / kBlock;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const int64_t r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
  float a = 0.f, d = 0.f;
  if (c < C) {
    for (int64_t r = r0 + warp; r < r1; r += 8) {
      const float fg = Elem<E>::widen1(g[r * C + c]);
      a = fmaf(fg, (input1<E, FMT>(x, scales, r, c, C, nb) - mean[r]) * rstd[r], a);
      d += fg;
    }
  }
  acc[0][warp][lane] = a;
  acc[1][warp][lane] = d;
  __syncthreads();
  if (warp < 2 && c < C) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += acc[warp][i][lane];
    part[(int64_t(blockIdx.y) * 2 + warp) * C + c] = s;
  }
}

// ------------------------------------------------------------------ launchers
// Team and chunks per lane for a width the register kernels take.
struct Shape {
  int team, nv, teams;
};
bool register_shape(int C, Shape *p) {
  if (C % 8 || C > 256 * kMaxNV * kMaxTeam) return false;
  const int warps = (C + 255) / 256;  // 256 values per warp and chunk
  p->team = 1;
  while (p->team * kMaxNV < warps) p->team *= 2;
  p->nv = (warps + p->team - 1) / p->team;
  if (p->nv == 3) p->nv = 4;
  p->teams = kWarps / p->team;
  return true;
}

#define FMHC_DISPATCH_NV(NV_RT, ...)                        \
  do {                                                      \
    if ((NV_RT) == 1) { constexpr int NV = 1; __VA_ARGS__; } \
    else if ((NV_RT) == 2) { constexpr int NV = 2; __VA_ARGS__; } \
    else { constexpr int NV = 4; __VA_ARGS__; }             \
  } while (0)
#define FMHC_DISPATCH_FMT_OR_NONE(FMT_RT, ...)                                  \
  do {                                                                          \
    if ((FMT_RT) == kNone) { constexpr int FMT = kNone; __VA_ARGS__; }          \
    else FMHC_DISPATCH_FMT(FMT_RT, __VA_ARGS__);                                \
  } while (0)

int sm_count() {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms > 0 ? sms : 1;
}

// Blocks of the register backward: at most two per SM, no more than the rows.
int bwd_blocks(int64_t rows, const Shape &p) {
  const int64_t need = (rows + p.teams - 1) / p.teams;
  const int64_t cap = std::min<int64_t>(2 * sm_count(), kMaxParts);
  return int(need < cap ? need : cap);
}
int any_slices(int64_t rows, int C) {
  const int64_t cols = (C + 31) / 32;
  int64_t n = (8 * int64_t(sm_count()) + cols - 1) / cols;
  n = std::min<int64_t>(n, (rows + 31) / 32);
  return int(std::min<int64_t>(std::max<int64_t>(n, 1), kMaxParts));
}

}  // namespace

void launch_ln_fwd(const void *x, int dtype, const void *w, const void *b, int pdt, float eps,
                   void *y, float *mean, float *rstd, void *codes, int fmt, void *scales,
                   int64_t rows, int C, bool vec, cudaStream_t s) {
  Shape p;
  if (vec && register_shape(C, &p)) {
    FMHC_DISPATCH_ELEM(dtype, FMHC_DISPATCH_FMT_OR_NONE(fmt, FMHC_DISPATCH_NV(p.nv, {
      auto k = ln_fwd_kernel<E, NV, FMT>;
      launch(k, dim3(grid_for(k, rows * p.team, kThreads)), dim3(kThreads), 0, s, (const E *)x, w,
             b, pdt, eps, (E *)y, mean, rstd, (uint8_t *)codes, (uint8_t *)scales, rows, C, p.team);
    })));
  } else {
    FMHC_DISPATCH_ELEM(dtype, FMHC_DISPATCH_FMT_OR_NONE(fmt, {
      auto k = ln_fwd_any_kernel<E, FMT>;
      launch(k, dim3(grid_for(k, rows * (kWarps), kThreads)), dim3(kThreads), 0, s,
             (const E *)x, w, b, pdt, eps, (E *)y, mean, rstd, (uint8_t *)codes, (uint8_t *)scales,
             rows, C);
    }));
  }
}

int64_t ln_bwd_workspace_bytes(int64_t rows, int C) {
  if (rows < 1 || C < 1) return 0;
  // The larger of the two paths, so that the size does not depend on alignment.
  Shape p;
  int64_t n = any_slices(rows, C);
  if (register_shape(C, &p)) n = std::max<int64_t>(n, bwd_blocks(rows, p));
  return (n * 2 * C * 4 + 255) & ~int64_t(255);
}

void launch_ln_bwd(const void *g, int dtype, const void *x, int fmt, const void *scales,
                   const float *mean, const float *rstd, const void *w, int pdt, void *gx, void *gw,
                   void *gb, float *ws, int64_t rows, int C, bool vec, cudaStream_t s) {
  Shape p;
  float *part = gw != nullptr || gb != nullptr ? ws : nullptr;
  int parts = 0;
  if (vec && register_shape(C, &p)) {
    parts = bwd_blocks(rows, p);
    const size_t smem = part != nullptr && p.teams > 1 ? size_t(2) * C * 4 : 0;
    FMHC_DISPATCH_ELEM(dtype, FMHC_DISPATCH_FMT_OR_NONE(fmt, FMHC_DISPATCH_NV(p.nv, {
      auto k = ln_bwd_kernel<E, NV, FMT>;
      launch(k, dim3(parts), dim3(kThreads), smem, s, (const E *)g, x, (const uint8_t *)scales,
             mean, rstd, w, pdt, (E *)gx, part, rows, C, p.team);
    })));
  } else {
    FMHC_DISPATCH_ELEM(dtype, FMHC_DISPATCH_FMT_OR_NONE(fmt, {
      auto k = ln_bwd_any_kernel<E, FMT>;
      launch(k, dim3(grid_for(k, rows * (kWarps), kThreads)), dim3(kThreads), 0, s,
             (const E *)g, x, (const uint8_t *)scales, mean, rstd, w, pdt, (E *)gx, rows, C);
      if (part != nullptr) {
        parts = any_slices(rows, C);
        launch(ln_param_part_any_kernel<E, FMT>, dim3((C + 31) / 32, parts), dim3(256), 0, s,
               (const E *)g, x, (const uint8_t *)scales, mean, rstd, part, rows, C);
      }
    }));
  }
  if (part != nullptr)
    launch(ln_param_grad_kernel, dim3((C + 31) / 32), dim3(256), 0, s, (const float *)part, gw, gb,
           pdt, parts, C);
}

}  // namespace fmhc
