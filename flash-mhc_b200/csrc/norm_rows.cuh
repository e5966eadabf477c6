// What the norms over rows share: parameters in their own type, sums over the
// lanes and warps that hold a row, chunks of eight values in shared memory, and
// the split of rows over teams of warps.
#pragma once

#include <algorithm>

#include "act8.cuh"
#include "grid.cuh"
#include "lane_ring.cuh"

namespace fmhc {
namespace norm_rows {

using namespace act8;

constexpr int kMaxTeam = 16;  // warps per row

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

// Sum of the values of `team` lanes (a power of two), of which every group of
// that many lanes has a copy.
__device__ __forceinline__ float group_sum(float v, int team) {
  for (int o = team >> 1; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
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
  if (lane == 0) slot[warp] = v;
  named_bar_sync(1 + warp / team, team * 32);
  const float2 o = slot[warp / team * team + (lane & (team - 1))];
  return make_float2(group_sum(o.x, team), group_sum(o.y, team));
}

// The warps of a row, any number up to 32 of them: what joining one value per warp
// needs, worked out once.  Slots and barriers as in team_sum.
struct Team {
  int size, first, bar, lane, span;  // warps; the first of them; barrier; lane; a power of two >= size
  __device__ __forceinline__ Team(int team, int warp, int lane_) {
    size = team;
    first = warp / team * team;
    bar = 1 + warp / team;
    lane = lane_;
    span = 1;
    while (span < team) span *= 2;
  }
  __device__ __forceinline__ int slot() const { return first + min(lane & (span - 1), size - 1); }
  __device__ __forceinline__ bool mine() const { return (lane & (span - 1)) < size; }
};
__device__ __forceinline__ float team_sum1(float v, float *slots, const Team &t, int warp) {
  if (t.size == 1) return v;
  if (t.lane == 0) slots[warp] = v;
  named_bar_sync(t.bar, t.size * 32);
  const float o = slots[t.slot()];
  return group_sum(t.mine() ? o : 0.f, t.span);
}
__device__ __forceinline__ uint32_t team_max(uint32_t v, uint32_t *slots, const Team &t, int warp) {
  if (t.size == 1) return v;
  if (t.lane == 0) slots[warp] = v;
  named_bar_sync(t.bar, t.size * 32);
  return __reduce_max_sync(0xffffffffu, slots[t.slot()]);
}

// Pairs of a chunk's eight values.
template <class E>
__device__ __forceinline__ void widen2(const typename Elem<E>::Raw &r, float2 (&f)[4]) {
  float v[8];
  Elem<E>::widen(r, v);
#pragma unroll
  for (int k = 0; k < 4; ++k) f[k] = make_float2(v[2 * k], v[2 * k + 1]);
}
__device__ __forceinline__ void param8x2(const void *p, int dtype, int c, float def, float2 (&f)[4]) {
  float v[8];
  param8(p, dtype, c, def, v);
#pragma unroll
  for (int k = 0; k < 4; ++k) f[k] = make_float2(v[2 * k], v[2 * k + 1]);
}
// One raw chunk of eight values to and from shared memory.
template <class E, int OFF>
__device__ __forceinline__ void copy_raw(uint32_t dst, const E *src) {
  copy_async_at<16, OFF>(dst, src);
  if constexpr (sizeof(E) == 4) copy_async_at<16, OFF + 16>(dst, src + 4);
}
template <class E, int OFF>
__device__ __forceinline__ typename Elem<E>::Raw load_raw(uint32_t a) {
  if constexpr (sizeof(E) == 4) return {load_shared16<OFF>(a), load_shared16<OFF + 16>(a)};
  else return load_shared16<OFF>(a);
}

// Columns of weight or bias kept in shared memory as f32, the first four values
// of every chunk and then the last four, so that neighbouring lanes read
// neighbouring words.
__device__ __forceinline__ void keep_param(float4 *dst, const void *p, int dtype, float def, int nchunk) {
  for (int c = threadIdx.x; c < nchunk; c += blockDim.x) {
    float f[8];
    param8(p, dtype, c, def, f);
    dst[c] = make_float4(f[0], f[1], f[2], f[3]);
    dst[nchunk + c] = make_float4(f[4], f[5], f[6], f[7]);
  }
}
// Chunk of a lane whose first chunk is at `lo` (first halves) and `hi`, I * 32
// chunks on.
template <int I>
__device__ __forceinline__ void kept_param(uint32_t lo, uint32_t hi, float (&f)[8]) {
  const uint4 a = load_shared16<I * 512>(lo), b = load_shared16<I * 512>(hi);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = __uint_as_float(w[k]);
}
template <int I>
__device__ __forceinline__ void kept_param(uint32_t lo, uint32_t hi, float2 (&f)[4]) {
  float v[8];
  kept_param<I>(lo, hi, v);
#pragma unroll
  for (int k = 0; k < 4; ++k) f[k] = make_float2(v[2 * k], v[2 * k + 1]);
}

// A parameter's gradient in the parameters' type.
__device__ __forceinline__ void store_param(void *p, int dtype, int c, float v) {
  if (p == nullptr) return;
  if (dtype == 0) reinterpret_cast<float *>(p)[c] = v;
  else if (dtype == 1) reinterpret_cast<__nv_bfloat16 *>(p)[c] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half *>(p)[c] = __float2half_rn(v);
}

// Team and chunks per lane for a width the register kernels take, and the teams
// per block: as many as keep every SM busy, so that few rows spread over the
// SMs and many rows fill them.
struct Shape {
  int team, nv, teams, threads;
  int64_t sums() const { return int64_t(team) * nv * 16 * 32; }  // of a block's partial
};
inline bool register_shape(int64_t rows, int C, int max_nv, int max_warps, Shape *p) {
  if (C % 8 || C > 256 * max_nv * kMaxTeam) return false;
  const int chunks = (C + 255) / 256;  // 256 values per warp and chunk
  p->team = 1;
  while (p->team * max_nv < chunks) p->team *= 2;
  p->nv = (chunks + p->team - 1) / p->team;
  if (p->nv == 3) p->nv = 4;
  const int64_t want = (rows + sm_count() - 1) / sm_count();
  p->teams = int(std::min<int64_t>(std::max<int64_t>(want, 1), max_warps / p->team));
  p->threads = p->teams * p->team * 32;
  return true;
}
inline int blocks_for(int64_t rows, const Shape &p) {
  return int(std::min<int64_t>((rows + p.teams - 1) / p.teams, sm_count()));
}

}  // namespace norm_rows
}  // namespace fmhc
