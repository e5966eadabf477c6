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
// One pass over the data: a team of 1..16 warps holds a row, NV chunks of eight
// values per lane, so x is read once forward, and x and g once backward.
// Backward, a lane keeps the same columns for every row its team takes, so its
// share of grad_w and grad_b stays in registers until the end; blocks write one
// partial each, and a small kernel adds the partials in block order (no
// atomics: the same bits every time).  Registers for those sums leave at most
// 16 warps per SM, too few to cover HBM's latency with loads into registers
// (a first version ran at a third of the copy rate), so the next rows are
// prefetched into a shared-memory ring (lane_ring.cuh).
//
// Measured, us (floor of the bytes at the copy rate): 65536 x 2048 bf16 forward
// 87-90 (82), backward 128-134 (123); 131072 x 1024 97-100 (82), 144 (123); with
// int8 codes 131072 x 1024 forward 113-124 (103), backward 131 (103); e4m3 codes,
// f16, 16384 x 4096 65 (52), 81 (52).  Memory bounds the plain ones; those with
// codes are bound by instructions (23 per value forward, 25 backward), and a
// backward ends with 8 us of joining the parameters' partials.
#include "fmhc_launch.h"
#include "norm_rows.cuh"

namespace fmhc {

using namespace act8;
using namespace norm_rows;

namespace {

// Warps per block, one block per SM.  Forward (65536 x 2048 / 16384 x 8192 bf16,
// 16384 x 4096 f16 with e4m3 codes, us): 24 90 / 99 / 65, 16 93 / 113 / 70, 20
// 92 / 121 / 67, 28 91 / 99 / 73.  Backward: 16, for 128 registers a thread.
constexpr int kFwdWarps = 24;
constexpr int kBwdWarps = 16;
constexpr int kThreads = 256;         // of the kernels for any width
constexpr int kWarps = kThreads / 32;
constexpr int kMaxParts = 1024;

constexpr int kStages = 3;  // ring depth in rows
// Most chunks per lane: the backward's sums take 16 registers per chunk, and
// f32 rows take twice the ring.
template <class E> constexpr int kMaxNV = sizeof(E) == 2 ? 4 : 2;

// -------------------------------------------------------------------- forward
// Scalar arithmetic: packed pairs, as in the backward, were no faster without
// and slower with the 8-bit copy (131072 x 1024: 98.5 against 100.2 us, with
// int8 113 against 125).
template <class E, int NV, int FMT>
__global__ void __launch_bounds__(32 * kFwdWarps, 1)
ln_fwd_kernel(const E *__restrict__ x, const void *__restrict__ w, const void *__restrict__ b,
              int pdt, float eps, E *__restrict__ y, float *__restrict__ mean_out,
              float *__restrict__ rstd_out, uint8_t *__restrict__ codes,
              uint8_t *__restrict__ scales, int64_t rows, int C, int team) {
  using Raw = typename Elem<E>::Raw;
  constexpr int S = kStages;
  extern __shared__ uint4 dyn[];
  __shared__ float2 slots[2][kFwdWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int teams = (blockDim.x >> 5) / team;
  const int wt = warp % team, first = warp - wt;
  const int nchunk = C / 8, nb = (C + kBlock - 1) / kBlock;
  constexpr int kChunk = 32 * int(sizeof(Raw));  // a warp's chunk in the ring
  const uint32_t ring = shared_addr(dyn) + warp * (S * NV * kChunk) + lane * int(sizeof(Raw));
  // Warp i of the team holds the NV * 32 chunks from i * NV * 32, those below
  // nchunk; this lane every 32nd, from c0: its chunk i exists if i * 32 < left.
  const auto count = [&](int i) { return min(max(nchunk - i * NV * 32, 0), NV * 32) * 8; };
  const int c0 = wt * NV * 32 + lane, left = nchunk - c0;
  const int mine = count(wt);
  // Lane i joins for warp i of the team, as does every lane `team` on.
  const float n_lane = float(count(lane & (team - 1))), inv_n = n_lane > 0.f ? 1.f / n_lane : 0.f;
  const float inv_mine = mine ? 1.f / float(mine) : 0.f, inv_C = 1.f / float(C);
  const int64_t step = int64_t(gridDim.x) * teams;
  int64_t r = int64_t(blockIdx.x) * teams + warp / team;
  pdl_wait();
  // Pointers that move on by one step of rows.
  const int64_t hop = step * C;
  const E *src = x + r * C + c0 * 8;
  E *dst = y + r * C + c0 * 8;
  uint8_t *code_dst = FMT == kNone ? nullptr : codes + r * C + c0 * 8;
  uint8_t *scale_dst = FMT == kNone ? nullptr : scales + r * nb + (c0 >> 2);
  int64_t fetched = r;
  const auto fetch = [&](int stage) {
    if (fetched < rows) {
      const uint32_t to = ring + stage * (NV * kChunk);
      unrolled<NV>([&](auto i) {
        if (i * 32 < left) copy_raw<E, i * kChunk>(to, src + i * 256);
      });
    }
    fetched += step;
    src += hop;
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s);
  float4 *ws = reinterpret_cast<float4 *>(reinterpret_cast<Raw *>(dyn) + (blockDim.x >> 5) * (S * NV * 32));
  float4 *bs = ws + 2 * nchunk;
  keep_param(ws, w, pdt, 1.f, nchunk);
  keep_param(bs, b, pdt, 0.f, nchunk);
  __syncthreads();
  const uint32_t w_lo = shared_addr(ws + c0), w_hi = shared_addr(ws + nchunk + c0);
  const uint32_t b_lo = shared_addr(bs + c0), b_hi = shared_addr(bs + nchunk + c0);
  int par = 0, stage = 0;
  for (; r < rows; r += step, par ^= 1) {
    fetch(stage == 0 ? S - 1 : stage - 1);
    copy_wait<S - 1>();
    float f[NV][8];
    uint32_t big[NV];  // largest magnitude of the chunk
    float s = 0.f;
    const uint32_t from = ring + stage * (NV * kChunk);
    unrolled<NV>([&](auto i) {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[i][k] = 0.f;
      big[i] = 0;
      if (i * 32 < left) {
        const Raw raw = load_raw<E, i * kChunk>(from);
        Elem<E>::widen(raw, f[i]);
        if constexpr (FMT != kNone) big[i] = amax8_raw<E>(raw);
      }
#pragma unroll
      for (int k = 0; k < 8; k += 2) s += f[i][k] + f[i][k + 1];
    });
    if (++stage == S) stage = 0;
    s = warp_sum(s);
    // (__fmul_rn: not to be contracted with the differences below, so that every
    // instantiation gives the same bits.)
    const float m_w = __fmul_rn(s, inv_mine);
    float q = 0.f, q1 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * 32 < left) {
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
          const float d = f[i][k] - m_w, d1 = f[i][k + 1] - m_w;
          q = fmaf(d, d, q);
          q1 = fmaf(d1, d1, q1);
        }
      }
    q = warp_sum(q + q1);
    float mean = m_w, m2 = q;
    if (team > 1) {
      // Join the warps: means first, then the squares about the row's mean.
      // One barrier per row: `slots` alternates (see team_sum).
      float2 *slot = slots[par] + first;
      if (lane == 0) slot[wt] = make_float2(s, q);
      named_bar_sync(1 + warp / team, team * 32);
      const float2 o = slot[lane & (team - 1)];
      mean = __fmul_rn(group_sum(o.x, team), inv_C);
      const float d = n_lane > 0.f ? fmaf(o.x, inv_n, -mean) : 0.f;
      m2 = group_sum(fmaf(n_lane * d, d, o.y), team);
    }
    const float rstd = rsqrtf(fmaf(m2, inv_C, eps));
    if (wt == 0 && lane == 0) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
    unrolled<NV>([&](auto i) {
      const bool in = i * 32 < left;
      if constexpr (FMT != kNone) {
        const uint32_t e = scale_byte<FMT>(amax_block(big[i]));
        if (in) {
          __stcs(reinterpret_cast<uint2 *>(code_dst + i * 256), encode8<FMT>(f[i], e));
          if ((lane & 3) == 0) __stcs(scale_dst + i * 8, uint8_t(e));
        }
      }
      if (in) {
        float fw[8], fb[8], o[8];
        kept_param<i>(w_lo, w_hi, fw);
        kept_param<i>(b_lo, b_hi, fb);
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = fmaf((f[i][k] - mean) * rstd, fw[k], fb[k]);
        st8(dst + i * 256, o);
      }
    });
    dst += hop;
    if constexpr (FMT != kNone) {
      code_dst += hop;
      scale_dst += step * nb;
    }
  }
}

// ------------------------------------------------------------------- backward
// A row's chunk of eight in the backward's ring: g, and x or its codes.
template <class E, int FMT> struct Input;
template <class E> struct Input<E, kNone> { using X = typename Elem<E>::Raw; };
template <class E> struct Input<E, kInt8> { using X = uint2; };
template <class E> struct Input<E, kE4m3> { using X = uint2; };
// mean and rstd, and NV * 2 + 1 words of scale bytes, to a multiple of 16.
template <int NV, int FMT>
constexpr int kRowBytes = FMT == kNone ? 16 : (8 + (NV * 2 + 1) * 4 + 15) / 16 * 16;

// x - mean of a chunk, from x (e unused) or from codes with scale byte e; off is
// -mean.  Rounded once (a code times its scale is exact), so that values near
// the mean keep their relative precision.
template <class E, int FMT>
__device__ __forceinline__ void centred(const typename Input<E, FMT>::X &raw, uint32_t e, float2 off,
                                        float2 (&d)[4]) {
  if constexpr (FMT == kNone) {
    widen2<E>(raw, d);
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = add2(d[i], off);
  } else {
    decode4x2<FMT>(raw.x, d[0], d[1]);
    decode4x2<FMT>(raw.y, d[2], d[3]);
    const float2 s = both(scale_value(e));
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = fma2(d[i], s, off);
  }
}

// The weight's columns of a lane come from shared memory as f32 (or, for rows
// whose weight does not fit there, from global memory) twice per row; holding
// them too would pass 128 registers.  For the same reason the second pass reads
// g and x from the ring again.
template <class E, int NV, int FMT, bool W_SHARED>
__global__ void __launch_bounds__(32 * kBwdWarps, 1)
ln_bwd_kernel(const E *__restrict__ g, const void *__restrict__ x,
              const uint8_t *__restrict__ scales, const float *__restrict__ mean,
              const float *__restrict__ rstd, const void *__restrict__ w, int pdt,
              E *__restrict__ gx, float *__restrict__ part, int64_t rows, int C, int team) {
  using Raw = typename Elem<E>::Raw;
  using X = typename Input<E, FMT>::X;
  constexpr int S = kStages;
  extern __shared__ uint4 dyn[];
  __shared__ float2 slots[2][kBwdWarps];
  const int warps = blockDim.x >> 5;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int teams = warps / team;
  const int wt = warp % team;
  const int nchunk = C / 8, nb = (C + kBlock - 1) / kBlock;
  const float inv_C = 1.f / float(C);
  // [warps][S][NV][32] of g, the same of x, then the weight.
  constexpr int kChunkG = 32 * int(sizeof(Raw)), kChunkX = 32 * int(sizeof(X));
  const uint32_t ring_g = shared_addr(dyn) + warp * (S * NV * kChunkG) + lane * int(sizeof(Raw));
  const uint32_t ring_x = shared_addr(dyn) + warps * (S * NV * kChunkG) + warp * (S * NV * kChunkX) +
                          lane * int(sizeof(X));
  // Per warp and row: mean and rstd, then the words that hold the scale bytes.  Unlike
  // the slots of g and x, a few lanes copy these for the whole warp, so a warp
  // barrier stands on both sides of a refill.
  const uint32_t ring_r = shared_addr(dyn) + warps * (S * NV * (kChunkG + kChunkX)) + warp * (S * kRowBytes<NV, FMT>);
  float4 *ws = reinterpret_cast<float4 *>(reinterpret_cast<char *>(dyn) + warps * (S * NV * (kChunkG + kChunkX)) +
                                          warps * (S * kRowBytes<NV, FMT>));
  const int64_t step = int64_t(gridDim.x) * teams;
  int64_t r = int64_t(blockIdx.x) * teams + warp / team;
  pdl_wait();
  // This lane's chunks: every 32nd of its warp's NV * 32, from c0 (as in the
  // forward); pointers that move on by one step of rows.
  const int c0 = wt * NV * 32 + lane, left = nchunk - c0;
  const int64_t hop = step * C;
  const E *g_src = g + r * C + c0 * 8;
  const E *x_src = FMT == kNone ? reinterpret_cast<const E *>(x) + r * C + c0 * 8 : nullptr;
  const uint8_t *q_src = FMT == kNone ? nullptr : reinterpret_cast<const uint8_t *>(x) + r * C + c0 * 8;
  E *dst = gx + r * C + c0 * 8;
  // Scale bytes of the warp's columns: from s_src on, wherever that lies in a word;
  // the words are copied (the last one up to the tensor's end).
  const uint8_t *s_src = FMT == kNone ? nullptr : scales + r * nb + wt * NV * 8;
  const uint8_t *const s_end = FMT == kNone ? nullptr : scales + rows * nb;
  int64_t fetched = r;
  const auto fetch = [&](int stage) {
    if (fetched < rows) {
      const uint32_t to_r = ring_r + stage * kRowBytes<NV, FMT>;
      if (lane >= 30) copy_async4(to_r + (lane - 30) * 4, (lane == 30 ? mean : rstd) + fetched);
      if constexpr (FMT != kNone) {
        const uint8_t *word = s_src - (reinterpret_cast<uintptr_t>(s_src) & 3) + 4 * lane;
        if (lane <= NV * 2 && word < s_end) copy_async4(to_r + 8 + lane * 4, word, int(min(s_end - word, int64_t(4))));
      }
      const uint32_t to_g = ring_g + stage * (NV * kChunkG), to_x = ring_x + stage * (NV * kChunkX);
      unrolled<NV>([&](auto i) {
        if (i * 32 < left) {
          copy_raw<E, i * kChunkG>(to_g, g_src + i * 256);
          if constexpr (FMT == kNone) copy_raw<E, i * kChunkX>(to_x, x_src + i * 256);
          else copy_async_at<8, i * kChunkX>(to_x, q_src + i * 256);
        }
      });
    }
    fetched += step;
    if constexpr (FMT != kNone) s_src += step * nb;
    g_src += hop;
    if constexpr (FMT == kNone) x_src += hop;
    else q_src += hop;
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s);
  if constexpr (W_SHARED) {
    keep_param(ws, w, pdt, 1.f, nchunk);
    __syncthreads();
  }
  const uint32_t w_lo = shared_addr(ws + c0), w_hi = shared_addr(ws + nchunk + c0);
  const auto weight = [&](auto i, float2 (&f)[4]) {
    if constexpr (W_SHARED) kept_param<i>(w_lo, w_hi, f);
    else param8x2(w, pdt, c0 + i * 32, 1.f, f);
  };
  const auto load_x = [&](auto i, uint32_t from) -> X {
    if constexpr (FMT == kNone) return load_raw<E, i * kChunkX>(from);
    else return load_shared8<i * kChunkX>(from);
  };
  float2 dw[NV][4], db[NV][4];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) dw[i][k] = db[i][k] = both(0.f);
  // Where this lane's scale byte of chunk 0 lies from its row's first word on:
  // s_src moves with the fetches, so the misalignment is followed separately.
  uint32_t s_off = FMT == kNone ? 0u : uint32_t(reinterpret_cast<uintptr_t>(scales + r * nb) & 3);
  int par = 0, stage = 0;
  for (; r < rows; r += step, par ^= 1) {
    __syncwarp();  // every lane has read the row slot that other lanes now refill
    fetch(stage == 0 ? S - 1 : stage - 1);
    copy_wait<S - 1>();
    __syncwarp();  // mean, rstd and scale bytes were copied by other lanes
    const uint32_t from_r = ring_r + stage * kRowBytes<NV, FMT>;
    const float2 stats = load_shared_f32x2(from_r);
    const float rs = stats.y;
    const float2 off = both(-stats.x);
    uint32_t e[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) e[i] = FMT == kNone ? 0u : load_shared_u8(from_r + 8 + s_off + (lane >> 2) + i * 8);
    s_off = (s_off + uint32_t(step * nb)) & 3u;
    float2 s1 = both(0.f), s2 = both(0.f);
    const uint32_t from_g = ring_g + stage * (NV * kChunkG), from_x = ring_x + stage * (NV * kChunkX);
    unrolled<NV>([&](auto i) {
      if (i * 32 < left) {
        float2 fg[4], d[4], fw[4];
        centred<E, FMT>(load_x(i, from_x), e[i], off, d);
        widen2<E>(load_raw<E, i * kChunkG>(from_g), fg);
        weight(i, fw);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 gw = mul2(fg[k], fw[k]), xh = mul2(d[k], both(rs));
          dw[i][k] = fma2(fg[k], xh, dw[i][k]);
          db[i][k] = add2(db[i][k], fg[k]);
          s1 = add2(s1, gw);
          s2 = fma2(gw, xh, s2);
        }
      }
    });
    const float2 sum = team_sum(make_float2(warp_sum(s1.x + s1.y), warp_sum(s2.x + s2.y)), slots[par],
                                team, warp, lane);
    const float2 c1 = both(-sum.x * inv_C), c2 = both(-sum.y * inv_C * rs);  // c2 times x - mean
    unrolled<NV>([&](auto i) {
      if (i * 32 < left) {
        float2 fg[4], d[4], fw[4];
        centred<E, FMT>(load_x(i, from_x), e[i], off, d);
        widen2<E>(load_raw<E, i * kChunkG>(from_g), fg);
        weight(i, fw);
        float o[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 v = mul2(both(rs), fma2(fg[k], fw[k], fma2(d[k], c2, c1)));
          o[2 * k] = v.x;
          o[2 * k + 1] = v.y;
        }
        st8(dst + i * 256, o);
      }
    });
    dst += hop;
    if (++stage == S) stage = 0;
  }
  if (part == nullptr) return;
  // Join the block's teams: every warp puts its sums into shared memory (the
  // ring's: no copy is in flight, since a row past the end fetches nothing, and
  // every warp has passed the barrier), then the block adds them in team order
  // and writes its partial.  A partial keeps the order of the lanes,
  // [wt][i * 8 + k, of grad_w then of grad_b][lane], so that all of this is
  // contiguous; ln_param_grad_kernel puts the columns in their places.
  constexpr int L = NV * 16 * 32;
  copy_wait<0>();
  __syncthreads();
  float *sums = reinterpret_cast<float *>(dyn);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      sums[warp * L + (i * 8 + k) * 32 + lane] = k & 1 ? dw[i][k / 2].y : dw[i][k / 2].x;
      sums[warp * L + ((NV + i) * 8 + k) * 32 + lane] = k & 1 ? db[i][k / 2].y : db[i][k / 2].x;
    }
  __syncthreads();
  float *out = part + int64_t(blockIdx.x) * team * L;
  for (int j = threadIdx.x; j < team * L; j += blockDim.x) {
    float v = 0.f;
    for (int t = 0; t < teams; ++t) v += sums[t * team * L + j];
    out[j] = v;
  }
}

// Adds n partials of `len` sums in a fixed order: grad_w and grad_b in the
// parameters' type.  Either may be absent.  nv 0: a partial is [2][C]; else it
// is in the lanes' order (see ln_bwd_kernel).  A block takes 32 sums; each of
// its 32 warps adds every 32nd partial, and the 32 results are added pairwise.
constexpr int kSumWarps = 32;
__global__ void __launch_bounds__(32 * kSumWarps)
ln_param_grad_kernel(const float *__restrict__ part, void *__restrict__ gw, void *__restrict__ gb,
                     int pdt, int n, int64_t len, int C, int nv) {
  pdl_wait();
  __shared__ float acc[kSumWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t j0 = int64_t(blockIdx.x) * 32;
  float a = 0.f;
  if (j0 + lane < len) {
#pragma unroll 8
    for (int i = warp; i < n; i += kSumWarps) a += part[i * len + j0 + lane];
  }
  acc[warp][lane] = a;
  __syncthreads();
  const float s = warp_sum(acc[lane][warp]);  // sum j0 + warp
  const int64_t j = j0 + warp;
  if (lane != 0 || j >= len) return;
  int c = int(j % C);
  bool is_b = j >= C;
  if (nv != 0) {
    const int l = int(j & 31);
    int q = int(j >> 5);  // (wt * 2 + which) * nv * 8 + i * 8 + k
    const int k = q & 7;
    q >>= 3;
    const int i = q % nv;
    q /= nv;
    is_b = q & 1;
    c = (((q >> 1) * nv + i) * 32 + l) * 8 + k;
    if (c >= C) return;
  }
  store_param(is_b ? gb : gw, pdt, c, s);
}

// ---------------------------------------------- any width and any alignment
// One block per row, which is read again for each step (from L1 or L2); forward, the
// first kKept values of each thread stay in registers.
constexpr int kKept = 4;
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
    float kept[kKept];
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
      const int c = i * kThreads + threadIdx.x;
      kept[i] = c < C ? Elem<E>::widen1(xr[c]) : 0.f;
    }
    // f(column, value) for this thread's columns.
    const auto each = [&](auto f) {
#pragma unroll
      for (int i = 0; i < kKept; ++i)
        if (i * kThreads + threadIdx.x < C) f(i * kThreads + int(threadIdx.x), kept[i]);
      for (int c = kKept * kThreads + threadIdx.x; c < C; c += kThreads) f(c, Elem<E>::widen1(xr[c]));
    };
    float2 v = make_float2(0.f, 0.f);
    each([&](int, float f) { v.x += f; });
    const float mean = block_sum(v, sh).x / float(C);
    v = make_float2(0.f, 0.f);
    each([&](int, float f) {
      const float d = f - mean;
      v.x = fmaf(d, d, v.x);
    });
    const float rstd = rsqrtf(block_sum(v, sh).x / float(C) + eps);
    if (threadIdx.x == 0) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
    each([&](int c, float f) {
      y[r * C + c] = Elem<E>::narrow1(fmaf((f - mean) * rstd, param1(w, pdt, c, 1.f), param1(b, pdt, c, 0.f)));
    });
    if constexpr (FMT != kNone) {
      for (int k = threadIdx.x >> 5; k < nb; k += kWarps) {  // a warp per block of 32
        const int c = k * kBlock + lane;
        const float f = c < C ? Elem<E>::widen1(xr[c]) : 0.f;
        const uint32_t e = scale_byte<FMT>(
            __reduce_max_sync(0xffffffffu, __float_as_uint(f) & 0x7fffffffu));
        if (c < C) codes[r * C + c] = encode1<FMT>(f, e);
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

// Any width up to 32 NV, a warp per row and the row in registers, 32 values apart
// in a lane: value i of the lanes is block i of 32.
template <class E, int FMT, int NV>
__global__ void __launch_bounds__(kThreads)
ln_fwd_warp_kernel(const E *__restrict__ x, const void *__restrict__ w, const void *__restrict__ b,
                   int pdt, float eps, E *__restrict__ y, float *__restrict__ mean_out,
                   float *__restrict__ rstd_out, uint8_t *__restrict__ codes,
                   uint8_t *__restrict__ scales, int64_t rows, int C) {
  pdl_wait();
  const int nb = (C + kBlock - 1) / kBlock, lane = threadIdx.x & 31;
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  for (int64_t r = warp; r < rows; r += nwarps) {
    const E *xr = x + r * C + lane;
    float f[NV], s = 0.f, q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) f[i] = i * 32 + lane < C ? Elem<E>::widen1(xr[i * 32]) : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) s += f[i];
    const float mean = warp_sum(s) / float(C);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float d = i * 32 + lane < C ? f[i] - mean : 0.f;
      q = fmaf(d, d, q);
    }
    const float rstd = rsqrtf(warp_sum(q) / float(C) + eps);
    if (lane == 0) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
    uint32_t mine = 0;  // lane i's: the scale byte of block i
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = i * 32 + lane;
      if (c < C)
        y[r * C + c] = Elem<E>::narrow1(fmaf((f[i] - mean) * rstd, param1(w, pdt, c, 1.f), param1(b, pdt, c, 0.f)));
      if constexpr (FMT != kNone) {
        if (i * 32 < C) {
          const uint32_t e = scale_byte<FMT>(
              __reduce_max_sync(0xffffffffu, __float_as_uint(f[i]) & 0x7fffffffu));
          if (c < C) codes[r * C + c] = encode1<FMT>(f[i], e);
          if (lane == i) mine = e;
        }
      }
    }
    if constexpr (FMT != kNone) {
      if (lane < nb) scales[r * nb + lane] = uint8_t(mine);
    }
  }
}

template <class E, int FMT, int NV>
__global__ void __launch_bounds__(kThreads)
ln_bwd_warp_kernel(const E *__restrict__ g, const void *__restrict__ x,
                   const uint8_t *__restrict__ scales, const float *__restrict__ mean,
                   const float *__restrict__ rstd, const void *__restrict__ w, int pdt,
                   E *__restrict__ gx, int64_t rows, int C) {
  pdl_wait();
  const int nb = (C + kBlock - 1) / kBlock, lane = threadIdx.x & 31;
  const int64_t warp = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (int64_t(gridDim.x) * kThreads) >> 5;
  for (int64_t r = warp; r < rows; r += nwarps) {
    const float m = mean[r], rs = rstd[r];
    float gw[NV], xh[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = i * 32 + lane;
      gw[i] = c < C ? Elem<E>::widen1(g[r * C + c]) : 0.f;
      xh[i] = c < C ? input1<E, FMT>(x, scales, r, c, C, nb) : m;
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = i * 32 + lane;
      if (c < C) gw[i] *= param1(w, pdt, c, 1.f);
      xh[i] = (xh[i] - m) * rs;
      s1 += gw[i];
      s2 = fmaf(gw[i], xh[i], s2);
    }
    const float c1 = warp_sum(s1) / float(C), c2 = warp_sum(s2) / float(C);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * 32 + lane < C) gx[r * C + i * 32 + lane] = Elem<E>::narrow1(rs * (gw[i] - fmaf(xh[i], c2, c1)));
  }
}

// Partials of grad_w and grad_b: block (cols of 32, slice of rows); the gradients
// themselves if there is one slice.
template <class E, int FMT>
__global__ void __launch_bounds__(256)
ln_param_part_any_kernel(const E *__restrict__ g, const void *__restrict__ x,
                         const uint8_t *__restrict__ scales, const float *__restrict__ mean,
                         const float *__restrict__ rstd, float *__restrict__ part, void *gw,
                         void *gb, int pdt, int64_t rows, int C) {
  __shared__ float acc[2][8][32];
  pdl_wait();
  const int nb = (C + kBlock - 1) / kBlock;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const int64_t r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
  float a = 0.f, d = 0.f;
  if (c < C) {
#pragma unroll 4
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
    if (gridDim.y == 1) store_param(warp ? gb : gw, pdt, c, s);
    else part[(int64_t(blockIdx.y) * 2 + warp) * C + c] = s;
  }
}

// ------------------------------------------------------------------ launchers
#define FMHC_DISPATCH_NV(NV_RT, NV_MAX, ...)                 \
  do {                                                       \
    if ((NV_RT) == 1) { constexpr int NV = 1; __VA_ARGS__; } \
    else if ((NV_RT) == 2 || (NV_MAX) == 2) { constexpr int NV = 2; __VA_ARGS__; } \
    else { constexpr int NV = (NV_MAX); __VA_ARGS__; }       \
  } while (0)
#define FMHC_DISPATCH_FMT_OR_NONE(FMT_RT, ...)                                  \
  do {                                                                          \
    if ((FMT_RT) == kNone) { constexpr int FMT = kNone; __VA_ARGS__; }          \
    else FMHC_DISPATCH_FMT(FMT_RT, __VA_ARGS__);                                \
  } while (0)

// Rows of widths that the ring kernels do not take go one to a warp if there are
// many of them and they are narrow, else one to a block (us, warp / block:
// forward 512 x 129 3.1 / 2.5, 2048 x 129 3.3 / 5.4, 65536 x 129 27 / 131, 65536 x
// 1023 223 / 201; backward 65536 x 1023 327 / 456, 4096 x 1023 27 / 27).
constexpr int64_t kManyRows = 1024;
constexpr int kFwdRowInWarp = 512, kBwdRowInWarp = 1024;
#define FMHC_WARP_KERNEL(KERNEL, C)                                          \
  ((C) <= 128 ? KERNEL<E, FMT, 4> : (C) <= 256 ? KERNEL<E, FMT, 8> : KERNEL<E, FMT, 16>)

// Slices of 32 rows or more; up to 128 rows are one, which needs no kernel to add
// partials (backward of f32 rows of 1023, one slice / slices of 32, us: 37 rows
// 5.4 / 6.8, 128 rows 6.4 / 7.0, 256 rows 7.9 / 7.2).
int any_slices(int64_t rows, int C) {
  if (rows <= 128) return 1;
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
  if (vec && register_shape(rows, C, dtype == 0 ? kMaxNV<float> : kMaxNV<__half>, kFwdWarps, &p)) {
    FMHC_DISPATCH_ELEM(dtype, FMHC_DISPATCH_FMT_OR_NONE(fmt, FMHC_DISPATCH_NV(p.nv, kMaxNV<E>, {
      auto k = ln_fwd_kernel<E, NV, FMT>;
      const size_t smem = size_t(p.threads) * kStages * NV * sizeof(typename Elem<E>::Raw) + size_t(C) * 8;
      allow_smem(reinterpret_cast<const void *>(k), smem);
      launch(k, dim3(blocks_for(rows, p)), dim3(p.threads), smem, s, (const E *)x, w, b, pdt, eps,
             (E *)y, mean, rstd, (uint8_t *)codes, (uint8_t *)scales, rows, C, p.team);
    })));
  } else {
    FMHC_DISPATCH_ELEM(dtype, FMHC_DISPATCH_FMT_OR_NONE(fmt, {
      auto k = ln_fwd_any_kernel<E, FMT>;
      const bool in_warp = rows >= kManyRows && C <= kFwdRowInWarp;
      if (in_warp) k = FMHC_WARP_KERNEL(ln_fwd_warp_kernel, C);
      launch(k, dim3(grid_for(k, in_warp ? rows : rows * kWarps, kThreads)), dim3(kThreads), 0, s, (const E *)x, w, b,
             pdt, eps, (E *)y, mean, rstd, (uint8_t *)codes, (uint8_t *)scales, rows, C);
    }));
  }
}

int64_t ln_bwd_workspace_bytes(int64_t rows, int C) {
  if (rows < 1 || C < 1) return 0;
  // The largest of the paths, so that the size depends on neither the type nor
  // the alignment.
  Shape p;
  int64_t n = int64_t(any_slices(rows, C)) * 2 * C;
  for (int nv : {kMaxNV<float>, kMaxNV<__half>})
    if (register_shape(rows, C, nv, kBwdWarps, &p)) n = std::max(n, blocks_for(rows, p) * p.sums());
  return (n * 4 + 255) & ~int64_t(255);
}

void launch_ln_bwd(const void *g, int dtype, const void *x, int fmt, const void *scales,
                   const float *mean, const float *rstd, const void *w, int pdt, void *gx, void *gw,
                   void *gb, float *ws, int64_t rows, int C, bool vec, cudaStream_t s) {
  Shape p{};
  float *part = gw != nullptr || gb != nullptr ? ws : nullptr;
  int parts = 0, nv = 0;
  int64_t len = 2 * int64_t(C);
  if (vec && register_shape(rows, C, dtype == 0 ? kMaxNV<float> : kMaxNV<__half>,
                            kBwdWarps, &p)) {
    parts = blocks_for(rows, p);
    nv = p.nv;
    len = p.sums();
    FMHC_DISPATCH_ELEM(dtype, FMHC_DISPATCH_FMT_OR_NONE(fmt, FMHC_DISPATCH_NV(p.nv, kMaxNV<E>, {
      const size_t ring = size_t(p.threads) * kStages * NV *
                          (sizeof(typename Elem<E>::Raw) + sizeof(typename Input<E, FMT>::X)) +
                          size_t(p.threads / 32) * kStages * kRowBytes<NV, FMT>;
      // The ring's memory later holds the 64 NV bytes of sums of every thread.
      static_assert(kStages * (sizeof(typename Elem<E>::Raw) + sizeof(typename Input<E, FMT>::X)) >= 64,
                    "sums fit the ring");
      // The weight goes beside the ring where it fits: always but for the widest
      // rows (from 8512 on) whose x is kept as 16-bit values.
      const size_t with_w = ring + size_t(C) * 4;
      auto k = ln_bwd_kernel<E, NV, FMT, true>;
      size_t smem = with_w;
      if constexpr (FMT == kNone && sizeof(E) == 2 && NV == kMaxNV<E>) {
        if (with_w > kMaxSmem) {
          k = ln_bwd_kernel<E, NV, FMT, false>;
          smem = ring;
        }
      }
      allow_smem(reinterpret_cast<const void *>(k), smem);
      launch(k, dim3(parts), dim3(p.threads), smem, s, (const E *)g, x, (const uint8_t *)scales, mean,
             rstd, w, pdt, (E *)gx, part, rows, C, p.team);
    })));
  } else {
    FMHC_DISPATCH_ELEM(dtype, FMHC_DISPATCH_FMT_OR_NONE(fmt, {
      auto k = ln_bwd_any_kernel<E, FMT>;
      const bool in_warp = rows >= kManyRows && C <= kBwdRowInWarp;
      if (in_warp) k = C <= 512 ? FMHC_WARP_KERNEL(ln_bwd_warp_kernel, C) : ln_bwd_warp_kernel<E, FMT, 32>;
      launch(k, dim3(grid_for(k, in_warp ? rows : rows * kWarps, kThreads)), dim3(kThreads), 0, s, (const E *)g, x,
             (const uint8_t *)scales, mean, rstd, w, pdt, (E *)gx, rows, C);
      if (part != nullptr) {
        parts = any_slices(rows, C);
        launch(ln_param_part_any_kernel<E, FMT>, dim3((C + 31) / 32, parts), dim3(256), 0, s,
               (const E *)g, x, (const uint8_t *)scales, mean, rstd, part, gw, gb, pdt, rows, C);
      }
    }));
  }
  if (part != nullptr && (nv != 0 || parts > 1))
    launch(ln_param_grad_kernel, dim3(unsigned((len + 31) / 32)), dim3(32 * kSumWarps), 0, s,
           (const float *)part, gw, gb, pdt, parts, len, C, nv);
}

}  // namespace fmhc
