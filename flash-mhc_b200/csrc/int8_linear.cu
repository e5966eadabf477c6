// Linear layer from 8-bit rows (rows8.cuh) on the 5th-generation tensor cores:
//
//   y[t, n] = xs[t] (ws[n] sum_k xc[t, k] wc[n, k]) + b[n]
//
// The sum of products is a whole number and exact (K < 2^17 keeps it within 32 bits,
// whatever the order).  Rounded to f32: the sum (beyond 2^24), its product with ws, and
// that times xs plus b, once; then y to its type.  The product of the two scales is not
// taken: it leaves f32's range where y does not (two scales of 1e-21, or a sum of 0 and
// scales of 1e20).  A sum times a weight's scale does only from weights of 2^104 on.
//
// The weight is the MMA's A operand (M = output columns n) and the activations
// are B (N = rows t), so that a thread of the epilogue holds one output column of
// many rows: its weight scale and bias stay in registers, a row's scale is one
// shared-memory word for the warp, a warp's stores of a row are contiguous for any
// N and any alignment of y, and few rows of activations make a narrow tile instead
// of an empty one.  TMA fills K's and the tiles' ends with zeros.
//
// Two kernels: pairs of CTAs that keep 256 x 256 tiles in TMEM (many tiles), and
// clusters that split K of one 128 x tn tile each (few).  Every mbarrier wait is
// bounded (sm100_ptx.cuh); outputs that a kernel gave up on are NaN.
#include <cuda.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "act8.cuh"
#include "fmhc_launch.h"
#include "grid.cuh"
#include "lane_ring.cuh"
#include "rows8.cuh"
#include "sm100_ptx.cuh"
#include "tma_map.h"

namespace fmhc {

using namespace act8;
using namespace sm100;

namespace {

constexpr int kBK = 128;                // bytes of K per stage: one swizzle row
constexpr int kBM = 128;                // output columns per CTA
constexpr int kATile = kBM * kBK;       // 16 KiB
constexpr int kThreads = 192;           // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue
constexpr int kEpiThreads = 128;
constexpr int kPairEpiThreads = 256;    // of a pair's CTA: warps 2-9
constexpr int kMaxTn = 256;

struct Args {
  const float *xs, *ws;
  const void *bias;
  int bias_dtype;
  int64_t T, N;
  int K;
  int tn;   // rows t per tile
  int tiles_n, tiles_t;
};

__device__ __forceinline__ float bias1(const void *b, int dtype, int64_t n) {
  if (b == nullptr) return 0.f;
  if (dtype == 0) return reinterpret_cast<const float *>(b)[n];
  if (dtype == 1) return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(b)[n]);
  return __half2float(reinterpret_cast<const __half *>(b)[n]);
}

// One output, as every kernel here rounds it.
__device__ __forceinline__ float scaled(int sum, float ws, float xs, float b) {
  return fmaf(__fmul_rn(__int2float_rn(sum), ws), xs, b);
}

// 32 rows of a column: `rows` of them are stored, from y (row 0, this column) on.
// No branch stands between the rows of a whole chunk: one per row made each wait for
// the latency of its own arithmetic (tiles of 256 x 256 took 20 us each).  Two columns
// of a row per store, swapped between lanes, were slower (65536 x 1024 x 1024: 63.4
// against 67.6 us), and so were converting the sums by ordinary arithmetic (83 against
// 72 at the time) and row addresses from a multiplication or from a base that the warp
// shares (24973 x 10752 x 48: 224 and 233 against 175).
template <class E>
__device__ __forceinline__ void store_rows(const int (&v)[32], int rows, const float *xs, float ws, float b,
                                           E *y, int64_t N, bool in) {
  E o[32];
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    const float4 x = *reinterpret_cast<const float4 *>(xs + j);
    const float2 p0 = mul2(make_float2(__int2float_rn(v[j]), __int2float_rn(v[j + 1])), both(ws));
    const float2 p1 = mul2(make_float2(__int2float_rn(v[j + 2]), __int2float_rn(v[j + 3])), both(ws));
    const float2 f0 = fma2(p0, make_float2(x.x, x.y), both(b));
    const float2 f1 = fma2(p1, make_float2(x.z, x.w), both(b));
    o[j] = Elem<E>::narrow1(f0.x);
    o[j + 1] = Elem<E>::narrow1(f0.y);
    o[j + 2] = Elem<E>::narrow1(f1.x);
    o[j + 3] = Elem<E>::narrow1(f1.y);
  }
  if (rows >= 32) {
    if (in) {
#pragma unroll
      for (int j = 0; j < 32; ++j, y += N) *y = o[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j, y += N)
      if (in && j < rows) *y = o[j];
  }
}
// One column of a tile: `rows` rows from this warp's lanes of TMEM.  (Loading the next
// chunk ahead costs registers and was slower: 24973 x 10752 x 48 166 against 158 us.)
template <class E>
__device__ __forceinline__ void store_column(uint32_t tmem, int rows, const float *xs, float ws, float b,
                                             E *y, int64_t N, bool in) {
  for (int c = 0; c < rows; c += 32) {
    uint32_t v[32];
    tmem_ld_32x32b_x32(tmem + uint32_t(c), v);
    tmem_wait_ld();
    store_rows(reinterpret_cast<const int (&)[32]>(v), rows - c, xs + c, ws, b, y + c * N, N, in);
  }
}
template <class E>
__device__ __forceinline__ void store_nan(int rows, E *y, int64_t N, bool in) {
  for (int j = 0; j < rows; ++j, y += N)
    if (in) *y = Elem<E>::narrow1(__uint_as_float(0x7fc00000u));
}

// ------------------------------------------------------------- pairs of CTAs
constexpr int kPairStages = 6;
struct alignas(1024) PairSmem {
  uint8_t a[kPairStages][kATile];
  uint8_t b[kPairStages][kATile];  // half of the tile's rows t: at most 128
  alignas(16) float xs[2][kMaxTn];
  uint64_t full[kPairStages], empty[kPairStages];
  uint64_t tfull[2], tempty[2], mma_done;
  uint32_t tmem_base;
  int abort;
};

enum : unsigned { kSitePairEmpty = 0x201, kSitePairFull = 0x202, kSitePairTempty = 0x203,
                  kSitePairTfull = 0x204, kSitePairDrain = 0x205 };

// Tile `id` -> (column tile, row tile): groups of eight column tiles, all row tiles
// of a group before the next, so that what runs at one time shares its operands
// in L2.
constexpr int kGroup = 8;
__device__ __forceinline__ void tile_of(int64_t id, int tiles_n, int tiles_t, int *n, int *t) {
  const int64_t per = int64_t(kGroup) * tiles_t;
  const int g = int(id / per);
  const int first = g * kGroup, size = min(tiles_n - first, kGroup);
  const int64_t r = id - g * per;
  *n = first + int(r % size);
  *t = int(r / size);
}

// Persistent: pair p takes tiles p, p + pairs, ...  Barriers: `full` is the
// leader's and counts the bytes of both CTAs' copies; a commit arrives on `empty`
// and `tfull` of both; the epilogue warps of both arrive on the leader's `tempty`.
// LOSE_COPY (test hook only, as in k1_tc.cu): the first CTA arms its first stage's
// barrier but issues no copy for it, so the waits on that stage can only expire.
template <class E, bool LOSE_COPY = false>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(64 + kPairEpiThreads, 1)
int8_linear_pair_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                        E *__restrict__ y, const Args A) {
  extern __shared__ uint8_t smem_raw[];
  PairSmem &sm = *reinterpret_cast<PairSmem *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int *abort = &sm.abort;
  const uint32_t rank = cluster_ctarank();
  const int64_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int64_t tiles = int64_t(A.tiles_n) * A.tiles_t;
  const int nk = (A.K + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(smem_u32(&sm.full[s]), 1);
      mbar_init(smem_u32(&sm.empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&sm.tfull[b]), 1);
      mbar_init(smem_u32(&sm.tempty[b]), 16);
    }
    mbar_init(smem_u32(&sm.mma_done), 1);
    sm.abort = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_x);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&sm.tmem_base), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  cluster_sync_all();  // both CTAs' barriers exist
  const uint32_t tmem = sm.tmem_base;
  pdl_wait();

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      const int half = A.tn / 2;
      const uint32_t bytes = 2u * (kATile + uint32_t(half) * kBK);
      bool ok = true;
      for (int64_t id = pair; id < tiles && ok; id += pairs) {
        int tile_n, tile_t;
        tile_of(id, A.tiles_n, A.tiles_t, &tile_n, &tile_t);
        const int32_t n0 = tile_n * 2 * kBM + int32_t(rank) * kBM;
        const int32_t t0 = tile_t * A.tn + int32_t(rank) * half;
        for (int kb = 0; kb < nk; ++kb) {
          if (!mbar_wait_cluster(smem_u32(&sm.empty[stage]), phase ^ 1, abort, kSitePairEmpty)) { ok = false; break; }
          const uint32_t full = smem_u32(&sm.full[stage]);
          if (rank == 0) mbar_arrive_expect_tx(full, bytes);
          const uint32_t lead = mapa_shared(full, 0);
          if (!(LOSE_COPY && blockIdx.x == 0 && issued == 0)) {
            tma_load_2d_pair(smem_u32(sm.a[stage]), &tmap_w, lead, kb * kBK, n0);
            tma_load_2d_pair(smem_u32(sm.b[stage]), &tmap_x, lead, kb * kBK, t0);
          }
          ++issued;
          if (++stage == kPairStages) { stage = 0; phase ^= 1; }
        }
      }
      // Leave when the MMAs have used what was loaded: then the copies have landed, and no
      // commit arrives here any more.  After a wait that gave up, the leader's barriers
      // see the last copies of both CTAs land; the other CTA leaves after it (cluster
      // barrier below).
      const int n = issued < kPairStages ? issued : kPairStages;
      int s = stage;
      uint32_t ph = phase;
      for (int i = 0; i < n; ++i) {
        if (--s < 0) { s = kPairStages - 1; ph ^= 1; }
        ok = ok && mbar_wait_cluster(smem_u32(&sm.empty[s]), ph, abort, kSitePairEmpty);
        if (!ok && rank == 0) mbar_wait(smem_u32(&sm.full[s]), ph, abort, kSitePairDrain, true);
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = idesc_i8_s32(2 * kBM, A.tn);
      const uint64_t ad0 = smem_desc(smem_u32(sm.a[0]), 16, 1024, 2), bd0 = smem_desc(smem_u32(sm.b[0]), 16, 1024, 2);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int64_t id = pair; id < tiles && ok; id += pairs) {
        if (!mbar_wait_cluster(smem_u32(&sm.tempty[acc]), acc_phase ^ 1, abort, kSitePairTempty)) break;
        tc_fence_after();
        const uint32_t d = tmem + uint32_t(acc * 256);
        for (int kb = 0; kb < nk; ++kb) {
          if (!mbar_wait_cluster(smem_u32(&sm.full[stage]), phase, abort, kSitePairFull)) { ok = false; break; }
          tc_fence_after();
          const uint64_t ad = ad0 + uint64_t(stage * (kATile / 16)), bd = bd0 + uint64_t(stage * (kATile / 16));
#pragma unroll
          for (int k = 0; k < kBK / 32; ++k)  // 32 bytes of K on: 2 in the descriptors' units
            mma_i8_ss_pair(d, ad + 2 * k, bd + 2 * k, idesc, (kb | k) != 0);
          mma_commit_pair(smem_u32(&sm.empty[stage]));
          if (++stage == kPairStages) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        mma_commit_pair(smem_u32(&sm.tfull[acc]));
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
      // All MMAs issued by this thread complete before TMEM is freed.
      mma_commit_pair_here(smem_u32(&sm.mma_done));
      mbar_wait(smem_u32(&sm.mma_done), 0, abort, kSitePairDrain, true);
    }
  } else {
    // Warp w of eight: the lanes of quarter w % 4 and half of the rows.  What a tile
    // needs from global memory is loaded while the one before is stored.
    const int q = warp & 3, me = int(threadIdx.x) - 64, half = A.tn / 2, h0 = warp < 6 ? 0 : half;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    int64_t n = 0, t0 = 0;
    int rows = 0;
    float ws = 0.f, b = 0.f, x = 0.f;
    const auto next = [&](int64_t id) {
      if (id >= tiles) return;
      int tile_n, tile_t;
      tile_of(id, A.tiles_n, A.tiles_t, &tile_n, &tile_t);
      n = int64_t(tile_n) * 2 * kBM + rank * kBM + q * 32 + lane;
      t0 = int64_t(tile_t) * A.tn;
      rows = int(min(A.T - t0, int64_t(A.tn)));
      ws = n < A.N ? A.ws[n] : 0.f;
      b = n < A.N ? bias1(A.bias, A.bias_dtype, n) : 0.f;
      x = me < rows ? A.xs[t0 + me] : 0.f;
    };
    next(pair);
    for (int64_t id = pair; id < tiles; id += pairs) {
      // This buffer was last read two tiles ago, before the barrier of the tile between.
      sm.xs[acc][me] = x;
      named_bar_sync(1, kPairEpiThreads);
      const float w0 = ws, b0 = b;
      const bool in = n < A.N;
      const int mine = min(rows - h0, half);
      E *const to = y + (t0 + h0) * A.N + n;
      next(id + pairs);
      ok = ok && mbar_wait_cluster(smem_u32(&sm.tfull[acc]), acc_phase, abort, kSitePairTfull);
      ok = __all_sync(0xffffffffu, ok);  // the loads below take whole warps
      if (!ok) {
        store_nan(mine, to, A.N, in);
        acc ^= 1;  // the scales of the rows still go where the other warps read them
        continue;
      }
      tc_fence_after();
      store_column(tmem + (uint32_t(q * 32) << 16) + uint32_t(acc * 256 + h0), mine, sm.xs[acc] + h0, w0, b0, to, A.N, in);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cta_remote(mapa_shared(smem_u32(&sm.tempty[acc]), 0));
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // nothing arrives at the other CTA any more
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ------------------------------------------------------- clusters that split K
// A cluster of S CTAs takes one tile of 128 columns and tn rows; CTA r runs the
// stages [r nk / S, (r + 1) nk / S).  Each thread of the epilogue stores its column's
// partial sums into the shared memory of the CTAs that finish the rows (row t: CTA
// t mod S), and after a cluster barrier those add them: stores do not wait for an
// answer, where loading the others' sums after the barrier took 1.5 us for 16 rows and
// 5 for 128.
struct SplitTail {
  uint64_t full[16], empty[16];
  uint64_t tfull;
  alignas(16) float xs[kMaxTn];
  uint32_t tmem_base;
  int abort;
  int bad;  // a CTA of the cluster gave up
};

enum : unsigned { kSiteSplitEmpty = 0x211, kSiteSplitFull = 0x212, kSiteSplitTfull = 0x214,
                  kSiteSplitDrain = 0x215 };

template <class E, int S, bool LOSE_COPY = false>
__global__ void __launch_bounds__(kThreads)
int8_linear_split_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                         E *__restrict__ y, const Args A, int stages, int tmem_cols) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *const base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stage_bytes = kATile + A.tn * kBK;
  SplitTail &sm = *reinterpret_cast<SplitTail *>(base + stages * stage_bytes);
  int *const part = reinterpret_cast<int *>(&sm + 1);  // S > 1: [S][tn / S, rounded up][128]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int *abort = &sm.abort;
  const uint32_t rank = S > 1 ? cluster_ctarank() : 0u;
  const int64_t id = blockIdx.x / unsigned(S);
  const int tile_n = int(id % A.tiles_n), tile_t = int(id / A.tiles_n);
  const int nk = (A.K + kBK - 1) / kBK;
  const int kb0 = int(rank) * nk / S, kb1 = (int(rank) + 1) * nk / S;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(smem_u32(&sm.full[s]), 1);
      mbar_init(smem_u32(&sm.empty[s]), 1);
    }
    mbar_init(smem_u32(&sm.tfull), 1);
    sm.abort = 0;
    sm.bad = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_x);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&sm.tmem_base), uint32_t(tmem_cols));
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (S > 1) cluster_sync_all();  // every CTA has started, and its `bad` is 0
  const uint32_t tmem = sm.tmem_base;
  pdl_wait();

  const int q = warp & 3;
  const int64_t n = int64_t(tile_n) * kBM + q * 32 + lane;
  const int64_t t0 = int64_t(tile_t) * A.tn;
  const int rows = int(min(A.T - t0, int64_t(A.tn)));
  const bool in = n < A.N;
  float ws = 0.f, b = 0.f;

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(smem_u32(&sm.empty[stage]), phase ^ 1, abort, kSiteSplitEmpty)) break;
        const uint32_t full = smem_u32(&sm.full[stage]);
        mbar_arrive_expect_tx(full, uint32_t(stage_bytes));
        const uint32_t a = smem_u32(base) + uint32_t(stage * stage_bytes);
        if (!(LOSE_COPY && blockIdx.x == 0 && issued == 0)) {
          tma_load_2d(a, &tmap_w, full, kb * kBK, tile_n * kBM);
          tma_load_2d(a + kATile, &tmap_x, full, kb * kBK, int32_t(t0));
        }
        ++issued;
        if (++stage == stages) { stage = 0; phase ^= 1; }
      }
      const int left = issued < stages ? issued : stages;
      for (int i = 0; i < left; ++i) {
        if (--stage < 0) { stage = stages - 1; phase ^= 1; }
        mbar_wait(smem_u32(&sm.full[stage]), phase, abort, kSiteSplitDrain, true);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = idesc_i8_s32(kBM, A.tn);
      const uint64_t ad0 = smem_desc(smem_u32(base), 16, 1024, 2);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(smem_u32(&sm.full[stage]), phase, abort, kSiteSplitFull)) break;
        tc_fence_after();
        const uint64_t ad = ad0 + uint64_t((stage * stage_bytes) >> 4), bd = ad + kATile / 16;
#pragma unroll
        for (int k = 0; k < kBK / 32; ++k) mma_i8_ss(tmem, ad + 2 * k, bd + 2 * k, idesc, kb > kb0 || k > 0);
        mma_commit(smem_u32(&sm.empty[stage]));
        if (++stage == stages) { stage = 0; phase ^= 1; }
      }
      // Also after a wait that gave up: everything issued is done before TMEM is freed.
      mma_commit(smem_u32(&sm.tfull));
      mbar_wait(smem_u32(&sm.tfull), 0, abort, kSiteSplitDrain, true);
    }
  } else {
    const int me = int(threadIdx.x) - 64;
    for (int i = me; i < rows; i += kEpiThreads) sm.xs[i] = A.xs[t0 + i];
    ws = in ? A.ws[n] : 0.f;
    b = in ? bias1(A.bias, A.bias_dtype, n) : 0.f;
    named_bar_sync(1, kEpiThreads);
    bool ok = mbar_wait(smem_u32(&sm.tfull), 0, abort, kSiteSplitTfull) && *abort == 0;
    ok = __all_sync(0xffffffffu, ok);  // the loads below take whole warps
    tc_fence_after();
    if constexpr (S == 1) {
      E *to = y + t0 * A.N + n;
      if (ok) store_column(tmem + (uint32_t(q * 32) << 16), rows, sm.xs, ws, b, to, A.N, in);
      else store_nan(rows, to, A.N, in);
    } else {
      const int each = (A.tn + S - 1) / S;
      uint32_t to[S];
#pragma unroll
      for (int s = 0; s < S; ++s)
        to[s] = mapa_shared(smem_u32(part + int(rank) * each * kBM + q * 32 + lane), uint32_t(s));
      if (ok) {
        for (int c = 0; c < rows; c += 32) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(tmem + (uint32_t(q * 32) << 16) + uint32_t(c), v);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c + j < rows) st_cluster_u32(to[j % S] + uint32_t((c + j) / S * kBM * 4), v[j]);
        }
      } else {
        for (uint32_t s = 0; s < S; ++s) st_cluster_u32(mapa_shared(smem_u32(&sm.bad), s), 1u);
      }
    }
  }
  tc_fence_before();
  if constexpr (S > 1) {
    __syncwarp();
    cluster_sync_all();  // the cluster's partial sums have arrived
    if (warp >= 2) {
      const int each = (A.tn + S - 1) / S;
      const bool ok = *reinterpret_cast<volatile int *>(&sm.bad) == 0;
      const int *from = part + q * 32 + lane;
      E *to = y + (t0 + rank) * A.N + n;
#pragma unroll 4
      for (int i = 0; int(rank) + i * S < rows; ++i) {
        int v = 0;
#pragma unroll
        for (int s = 0; s < S; ++s) v += from[(s * each + i) * kBM];
        const float f = ok ? scaled(v, ws, sm.xs[int(rank) + i * S], b) : __uint_as_float(0x7fc00000u);
        if (in) to[int64_t(i) * S * A.N] = Elem<E>::narrow1(f);
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, uint32_t(tmem_cols));
  }
}

// ------------------------------------------------------------ a handful of rows
// Up to four rows t read the weight once at the rate of memory, and dot products of
// four bytes on the CUDA cores keep up with it.  A warp takes kRowCols columns n and
// every `split`-th stretch of kRowBytes bytes of K per lane-wide load; its lanes' sums
// are added by the warp, and those of `split` warps in shared memory.
constexpr int kRowsMost = 4;
constexpr int kRowWarps = 4, kRowCols = 2, kRowDepth = 4;  // loads in flight: columns x depth

// 16 codes from k on, of which `there` are the row's own; zeros for the others.
__device__ __forceinline__ uint4 load_codes16(const int8_t *p, int there) {
  if (there >= 16) return __ldg(reinterpret_cast<const uint4 *>(p));
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int k = 0; k < 16; ++k)
    if (k < there) w[k >> 2] |= uint32_t(uint8_t(p[k])) << (8 * (k & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <class E, int TT>
__global__ void __launch_bounds__(32 * kRowWarps)
int8_linear_rows_kernel(const int8_t *__restrict__ xc, int64_t xstride, const int8_t *__restrict__ wc, int64_t wstride,
                        E *__restrict__ y, const Args A, int split) {
  __shared__ int sums[kRowWarps][kRowCols][TT];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n0 = (int64_t(blockIdx.x) * (kRowWarps / split) + warp / split) * kRowCols;
  const int T = int(A.T), K = A.K;
  pdl_wait();
  const int8_t *w[kRowCols];
#pragma unroll
  for (int c = 0; c < kRowCols; ++c) w[c] = wc + min(n0 + c, A.N - 1) * wstride;
  int acc[kRowCols][TT];
#pragma unroll
  for (int c = 0; c < kRowCols; ++c)
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[c][t] = 0;
  const int8_t *x[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) x[t] = xc + min(t, T - 1) * xstride;
  const auto add = [&](const uint4 &q, const uint4 (&v)[kRowCols], int t) {
#pragma unroll
    for (int c = 0; c < kRowCols; ++c) {
      acc[c][t] = __dp4a(int(q.x), int(v[c].x), acc[c][t]);
      acc[c][t] = __dp4a(int(q.y), int(v[c].y), acc[c][t]);
      acc[c][t] = __dp4a(int(q.z), int(v[c].z), acc[c][t]);
      acc[c][t] = __dp4a(int(q.w), int(v[c].w), acc[c][t]);
    }
  };
  constexpr int kStretch = 512 * kRowDepth;
  int k0 = (warp % split) * kStretch;
  for (; k0 + kStretch <= K; k0 += split * kStretch) {  // whole stretches: no branch between the loads
    const int k = k0 + lane * 16;
    uint4 v[kRowDepth][kRowCols];
#pragma unroll
    for (int d = 0; d < kRowDepth; ++d)
#pragma unroll
      for (int c = 0; c < kRowCols; ++c) v[d][c] = __ldg(reinterpret_cast<const uint4 *>(w[c] + k + d * 512));
#pragma unroll
    for (int d = 0; d < kRowDepth; ++d) {
      uint4 q[TT];
#pragma unroll
      for (int t = 0; t < TT; ++t) q[t] = __ldg(reinterpret_cast<const uint4 *>(x[t] + k + d * 512));
#pragma unroll
      for (int t = 0; t < TT; ++t) add(q[t], v[d], t);
    }
  }
  for (int k = k0 + lane * 16; k < min(K, k0 + kStretch); k += 512) {  // the last, shorter one
    uint4 v[kRowCols];
#pragma unroll
    for (int c = 0; c < kRowCols; ++c) v[c] = load_codes16(w[c] + k, K - k);
#pragma unroll
    for (int t = 0; t < TT; ++t) add(load_codes16(x[t] + k, K - k), v, t);
  }
#pragma unroll
  for (int c = 0; c < kRowCols; ++c)
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int v = __reduce_add_sync(0xffffffffu, acc[c][t]);
      if (lane == 0) sums[warp][c][t] = v;
    }
  __syncthreads();
  // One value per thread: column c of warp group `g`, row t.
  constexpr int kOut = kRowCols * TT;
  for (int i = threadIdx.x; i < kRowWarps / split * kOut; i += blockDim.x) {
    const int g = i / kOut, t = i / kRowCols % TT, c = i % kRowCols;
    const int64_t n = (int64_t(blockIdx.x) * (kRowWarps / split) + g) * kRowCols + c;
    if (t < T && n < A.N) {
      int v = 0;
      for (int k = 0; k < split; ++k) v += sums[g * split + k][c][t];
      y[t * A.N + n] = Elem<E>::narrow1(scaled(v, A.ws[n], A.xs[t], bias1(A.bias, A.bias_dtype, n)));
    }
  }
}

// ------------------------------------------------------------------ launchers
bool make_map(CUtensorMap *m, const void *base, int K, int64_t rows, int64_t stride, int box_rows) {
  const auto fn = encode_fn();
  if (fn == nullptr) return false;
  cuuint64_t dims[2] = {cuuint64_t(K), cuuint64_t(rows)};
  cuuint64_t strides[1] = {cuuint64_t(stride)};
  cuuint32_t box[2] = {kBK, cuuint32_t(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace

int read_int8_linear_error(unsigned *code) {
  unsigned v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, sm100::g_device_error, sizeof(v)) != cudaSuccess) return 5;
  if (v && cudaMemcpyToSymbol(sm100::g_device_error, &zero, sizeof(zero)) != cudaSuccess) return 5;
  *code = v;
  return 0;
}

int launch_int8_linear(const void *xc, int64_t xstride, const float *xs, const void *wc, int64_t wstride,
                       const float *ws, const void *b, int bdt, void *y, int ydt, int64_t T, int64_t N,
                       int K, cudaStream_t s, bool lose_copy) {
  const int sms = sm_count();
  const int nk = int(ceil_div(K, kBK));
  Args a{};
  a.xs = xs; a.ws = ws; a.bias = b; a.bias_dtype = bdt;
  a.T = T; a.N = N; a.K = K;
  // The kernel for a handful of rows is the faster one while its arithmetic is little
  // (us, it / tiles of 128 columns: T x N x K 1 x 4096 x 4096 5.4 / 6.7, 1 x 8192 x 4096
  // 7.2 / 8.9, 1 x 16384 x 4096 13.1 / 13.0; 2 x 2048 x 2048 2.3 / 3.8, 4 x 2048 x 2048
  // 3.1 / 3.9, 4 x 4096 x 1024 3.4 / 3.7, 2 x 2896 x 2896 5.8 / 5.7, 2 x 4096 x 4096
  // 7.1 / 6.6, 4 x 4096 x 2048 6.0 / 5.2).  For five rows and more the tiles are (an
  // instance for eight took 8 x 1024 x 1024 in 4.6 us, they 3.4; 5 x 3000 x 2200 11.4 / 5.1;
  // the only ones it was faster at are as small as 5 x 512 x 512, 2.5 / 2.8).
  if (!lose_copy && T <= kRowsMost && T * N * K <= int64_t(1) << (T == 1 ? 25 : 24)) {
    int split = 1;  // warps that share K: enough blocks for every SM, while there is K for them
    while (split < kRowWarps && ceil_div(N, kRowCols * (kRowWarps / split)) < 2 * sms && K > split * 512 * kRowDepth) split *= 2;
    const int64_t blocks = ceil_div(N, int64_t(kRowCols) * (kRowWarps / split));
    FMHC_DISPATCH_ELEM(ydt, {
      auto k = T == 1 ? int8_linear_rows_kernel<E, 1> : T == 2 ? int8_linear_rows_kernel<E, 2>
             : int8_linear_rows_kernel<E, kRowsMost>;
      launch(k, dim3(unsigned(blocks)), dim3(32 * kRowWarps), 0, s, (const int8_t *)xc, xstride, (const int8_t *)wc, wstride,
             (E *)y, a, split);
    });
    return 0;
  }
  CUtensorMap mw, mx;
  const int64_t pair_t = ceil_div(T, kMaxTn);
  // Pairs of CTAs once they keep three quarters of the SMs busy (us, pairs / tiles of
  // one CTA: 256 x 4096 x 4096 14.9 / 8.7, 1024 x 2048 x 2048 10.9 / 7.8, 512 x 4096 x
  // 4096 15.4 / 11.0, 1024 x 4096 x 4096 16.0 / 17.0, 512 x 16384 x 4096 26.9 / 36.2).
  if (ceil_div(N, 2 * kBM) * pair_t * 2 >= sms * 3 / 4 && T > 128) {
    a.tiles_t = int(pair_t);
    a.tn = int(ceil_div(ceil_div(T, pair_t), 32) * 32);
    a.tiles_n = int(ceil_div(N, 2 * kBM));
    if (!make_map(&mw, wc, K, N, wstride, kBM) || !make_map(&mx, xc, K, T, xstride, a.tn / 2))
      return set_last_error(5, "fmhc_int8_linear: cuTensorMapEncodeTiled failed");
    const int64_t pairs = std::min<int64_t>(int64_t(a.tiles_n) * a.tiles_t, sms / 2);
    const size_t smem = sizeof(PairSmem) + 1024;
    FMHC_DISPATCH_ELEM(ydt, {
      auto k = int8_linear_pair_kernel<E>;
      if constexpr (std::is_same<E, __nv_bfloat16>::value) {
        if (lose_copy) k = int8_linear_pair_kernel<E, true>;
      }
      allow_smem(reinterpret_cast<const void *>(k), smem);
      launch(k, dim3(unsigned(pairs * 2)), dim3(64 + kPairEpiThreads), smem, s, mw, mx, (E *)y, a);
    });
    return 0;
  }
  a.tiles_n = int(ceil_div(N, kBM));
  // Tiles of up to 128 rows, narrower ones (down to 32, or 64 for a long K) where that
  // gives more SMs one (us, as chosen / always 128: 100 x 4096 x 4096 8.0 / 10.2, 256 x
  // 4096 x 4096 8.8 / 10.9; 64 x 4096 x 16384 with tiles of 64 / of 32 15.7 / 16.8).
  const int least = nk >= 64 ? 64 : 32;
  int64_t tiles_t = std::max(ceil_div(T, 128), std::min<int64_t>(ceil_div(T, least), sms / a.tiles_n));
  a.tn = int(ceil_div(ceil_div(T, tiles_t), 16) * 16);
  a.tiles_t = int(ceil_div(T, a.tn));
  if (!make_map(&mw, wc, K, N, wstride, kBM) || !make_map(&mx, xc, K, T, xstride, a.tn))
    return set_last_error(5, "fmhc_int8_linear: cuTensorMapEncodeTiled failed");
  const int64_t tiles = int64_t(a.tiles_n) * a.tiles_t;
  if (tiles > (int64_t(1) << 27))
    return set_last_error(2, "fmhc_int8_linear: T and N give more than 2^27 tiles");
  // K is split where the stages that a CTA is spared (about 0.12 us each) outweigh the
  // cluster's exchange of partial sums, which grows with the tile (us, 1 / 2 / 4 CTAs: 16 x
  // 1024 x 1024 3.7 / 4.0 / 3.5, 16 x 4096 x 4096 7.8 / 7.5 / 6.9, 64 x 2048 x 2048 5.3 /
  // 5.6 / 5.0, 64 x 4096 x 16384 23 / 19 / 16), up to as many clusters as run at one time
  // (16 of eight CTAs do not: 16 x 2048 x 2048 7.1, of four 4.1).
  const int worth = 4 + a.tn / 5;
  const int S = tiles <= 8 && nk >= 2 * worth ? 8 : tiles <= 32 && nk >= worth ? 4 : tiles <= 64 && nk >= 2 * worth ? 2 : 1;
  int cols = 32;
  while (cols < a.tn) cols *= 2;
  const int stage_bytes = kATile + a.tn * kBK;
  const int part_bytes = S > 1 ? S * ((a.tn + S - 1) / S) * kBM * 4 : 0;
  const int stages = std::min(((tiles * S > sms ? 100 : 200) * 1024 - part_bytes) / stage_bytes, 12);
  const size_t smem = size_t(stages) * stage_bytes + sizeof(SplitTail) + part_bytes + 1024;
  FMHC_DISPATCH_ELEM(ydt, {
    auto k = S == 1 ? int8_linear_split_kernel<E, 1> : S == 2 ? int8_linear_split_kernel<E, 2>
           : S == 4 ? int8_linear_split_kernel<E, 4> : int8_linear_split_kernel<E, 8>;
    if constexpr (std::is_same<E, __nv_bfloat16>::value) {
      if (lose_copy)
        k = S == 1 ? int8_linear_split_kernel<E, 1, true> : S == 2 ? int8_linear_split_kernel<E, 2, true>
          : S == 4 ? int8_linear_split_kernel<E, 4, true> : int8_linear_split_kernel<E, 8, true>;
    }
    allow_smem(reinterpret_cast<const void *>(k), smem);
    launch_cluster(k, dim3(unsigned(tiles * S)), dim3(kThreads), smem, s, unsigned(S), mw, mx, (E *)y, a, stages, cols);
  });
  return 0;
}

}  // namespace fmhc
