// K1 backward on the tensor cores: grad_x and (optionally) grad_W in one pass
// over x.  Included by k1_tc.cu (same translation unit as the forward kernel,
// sharing its PTX helpers and device error word).
//
//   s[t]        = (sum_d go[t,d] proj[t,d]) * inv_rms[t]^2 / nC
//   grad_x[t,k] = bf16( inv_rms[t] * sum_d go[t,d] W[d,k] - s[t] * x[t,k] )
//   grad_W[d,k] = bf16( sum_t gos[t,d] x[t,k] ),  gos = bf16(go * inv_rms)
//
// (src/flash_mhc/kernels.py:306-376 and src/flash_mhc/ops.py:683-684 of the
// reference.)  Work unit = (k-chunk of 128 columns, tile of 128 tokens).
//
// Work order.  The k-chunks are split into groups of G (<= 8) and every
// persistent CTA belongs to one group for its whole life: CTA i of a group of
// ng CTAs takes the token tiles i, i + ng, i + 2 ng, ... and, for each tile,
// the group's G k-chunks in order.  So all CTAs sweep the tokens together (at
// any moment the whole GPU reads and writes a window of a few dozen token
// tiles, which keeps HBM pages and write-backs local), each x row is read
// G x 256 contiguous bytes per tile, and each CTA accumulates the grad_W
// partials of its G k-chunks in TMEM over all its tiles.
//
//   warp 0     TMA producer: per token tile go[128 t x 32] and proj[128 t x 32]
//              (64-byte swizzle) into a tile slot (two slots); per unit
//              x[128 t x 128 k] (two 64-column boxes, 128-byte swizzle) and the
//              W chunk [32 x 128 k] into a stage (four stages).
//   warp 1     MMA issuer, per unit:
//                grad_W: D2_j[k, d] += x^T (MN-major A) * gos (MN-major B),
//                        8 x M128 N32 K16 into accumulator j of the group;
//                grad_x: D1[t, k]  = go (K-major A) * W^T (MN-major B),
//                        2 x M128 N128 K16 into one of two TMEM buffers.
//   warps 2-9  epilogue, two warps per TMEM lane quarter: thread = token row,
//              warps 2-5 columns 0-63, warps 6-9 columns 64-127 of the unit:
//              grad_x = inv*D1 - s*x written over x in the stage buffer.  At
//              the end they move the G grad_W partials (thread per k row) to
//              the workspace.
//   warp 10    store: TMA-stores each unit's grad_x from its stage, keeps up to
//              two stores in flight and frees a stage as soon as its store has
//              read it.
//   warp 11    tile prep, once per token tile: (s, inv_rms) per token and the
//              grad_W operand gos = bf16(go * inv_rms) (same 64-byte swizzle
//              as go) into the slot, from the slot's go and proj and inv_rms.
// A final small kernel reduces the per-CTA grad_W partials of each group in a
// fixed order (deterministic) and rounds to bf16.  The grad_x-only variant
// runs the same kernel without the grad_W MMAs and needs no workspace.
#pragma once

#include "k1_bwd_plan.h"

namespace fmhc {
namespace k1tc {

#ifndef FMHC_K1B_STAGES
#define FMHC_K1B_STAGES 4
#endif
// grad_x TMA stores outstanding per CTA (1..3).  Measured at T=65536, nC=4096:
// 2 -> 174 us, 3 -> 216 us for the main kernel.
#ifndef FMHC_K1B_STORES_IN_FLIGHT
#define FMHC_K1B_STORES_IN_FLIGHT 2
#endif
static_assert(kBwdD == kND, "projection width");
constexpr int kBwdStages = FMHC_K1B_STAGES;
constexpr int kBwdInflight = FMHC_K1B_STORES_IN_FLIGHT;
static_assert(kBwdInflight >= 1 && kBwdInflight <= 3 && kBwdInflight < kBwdStages,
              "stores in flight");
constexpr int kBwdSlots = 2;                      // token-tile slots (go, proj, gos, (s, inv))
constexpr int kBwdXBytes = kBwdBT * kBwdBK * 2;   // 32 KiB (two 16 KiB boxes)
constexpr int kBwdXBox = kBwdBT * 64 * 2;         // 16 KiB
constexpr int kBwdWBytes = kND * kBwdBK * 2;      // 8 KiB  (two 4 KiB boxes)
constexpr int kBwdStageBytes = kBwdXBytes + kBwdWBytes;  // 40 KiB
constexpr int kBwdGBytes = kBwdBT * kND * 2;      // 8 KiB  (go, proj or gos tile)
constexpr int kBwdSBytes = kBwdBT * 8;            // 1 KiB  ((s, inv_rms) per token)
// Slot layout: go at 0, proj at 8 KiB (TMA), gos at 16 KiB, (s, inv) at 24 KiB (prep warp).
constexpr int kBwdSlotGo = 0, kBwdSlotProj = kBwdGBytes, kBwdSlotGos = 2 * kBwdGBytes,
              kBwdSlotSinv = 3 * kBwdGBytes;
constexpr int kBwdSlotBytes = 3 * kBwdGBytes + kBwdSBytes;  // 25 KiB
constexpr int kBwdThreads = 384;                  // producer, MMA, 8 epilogue warps, store, prep
constexpr int kBwdEpiWarps = 8;
constexpr int kBwdStoreWarp = 2 + kBwdEpiWarps;
constexpr int kBwdPrepWarp = kBwdStoreWarp + 1;
// Two 128-column grad_x accumulators, then up to 8 x 32 grad_W columns.
constexpr uint32_t kBwdTmemCols = 512;
constexpr uint32_t kBwdDwCol = 256;

struct alignas(1024) BwdSmem {
  uint8_t stage[kBwdStages][kBwdStageBytes];  // x tile, then the W chunk
  uint8_t slot[kBwdSlots][kBwdSlotBytes];     // go, proj, gos, (s, inv) of one token tile
  uint64_t full[kBwdStages];
  uint64_t empty[kBwdStages];
  // epi[s]: the 8 epilogue warps finished writing grad_x into stage s.  Its
  // next phase belongs to the next unit in that stage, which cannot be loaded
  // before the store warp has waited on this phase and freed the stage, so
  // phases never alias and each counts one unit's arrivals.
  uint64_t epi[kBwdStages];
  uint64_t gfull[kBwdSlots];   // go and proj landed
  uint64_t gready[kBwdSlots];  // prep warp wrote gos and (s, inv)
  uint64_t gempty[kBwdSlots];  // MMA commit after the tile's last unit + 8 epilogue warps
  uint64_t tfull[2];
  uint64_t tempty[2];
  uint64_t dwfull;
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort;
};

enum : unsigned { kSiteBProdEmpty = 0x201, kSiteBProdSlot = 0x202, kSiteBMmaFull = 0x203,
                  kSiteBMmaTempty = 0x204, kSiteBMmaSlot = 0x205, kSiteBEpiSlot = 0x206,
                  kSiteBEpiFull = 0x207, kSiteBEpiTfull = 0x208, kSiteBEpiDw = 0x209,
                  kSiteBDrain = 0x20a, kSiteBEpiStore = 0x20b, kSiteBPrepSlot = 0x20c };

struct BwdArgs {
  const float *inv_rms;       // (T,)
  float *dw_part;             // [grid][G][32][128] f32 (only with_dw)
  int64_t T;
  int nC;
  int ntt;                    // token tiles
  int G;                      // k-chunks per group
  int base, rem;              // CTAs per group: the first rem groups base + 1, the others base
  int with_dw;
};

// CTA c -> (group g, index i within the group, CTAs in the group ng).
__host__ __device__ __forceinline__ void bwd_cta_group(int c, int base, int rem, int &g, int &i,
                                                       int &ng) {
  const int big = rem * (base + 1);
  if (c < big) {
    g = c / (base + 1);
    i = c % (base + 1);
    ng = base + 1;
  } else {
    const int c2 = c - big;
    g = rem + c2 / base;
    i = c2 % base;
    ng = base;
  }
}
__host__ __device__ __forceinline__ int bwd_group_first_cta(int g, int base, int rem) {
  return g < rem ? g * (base + 1) : rem * (base + 1) + (g - rem) * base;
}

// Partial dot product of one 16-byte chunk (8 of the 32 d) of go and proj.
// The full dot product is (p0 + p1) + (p2 + p3) over the four chunks.
__device__ __forceinline__ float go_proj_chunk_dot(const uint4 g, const uint4 p) {
  float dot = 0.f;
  dot = fmaf(bf16lo(g.x), bf16lo(p.x), dot); dot = fmaf(bf16hi(g.x), bf16hi(p.x), dot);
  dot = fmaf(bf16lo(g.y), bf16lo(p.y), dot); dot = fmaf(bf16hi(g.y), bf16hi(p.y), dot);
  dot = fmaf(bf16lo(g.z), bf16lo(p.z), dot); dot = fmaf(bf16hi(g.z), bf16hi(p.z), dot);
  dot = fmaf(bf16lo(g.w), bf16lo(p.w), dot); dot = fmaf(bf16hi(g.w), bf16hi(p.w), dot);
  return dot;
}

// Tile prep of one slot by one warp: gos = bf16(go * inv_rms) and (s, inv_rms)
// per token, from the slot's go and proj.  Lane l takes the tile rows l, l + 32,
// l + 64, l + 96, whose inv_rms are invr.  GOS may be proj's own place: a chunk
// of gos is written after the chunk of proj there has been read.
template <int GOS, int SINV>
__device__ __forceinline__ void prep_tile(uint8_t *sb, int lane, const float (&invr)[4], float nC) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = lane + 32 * i;
    const float rinv = invr[i];
    float pc[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int off = r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
      const uint4 g = *reinterpret_cast<const uint4 *>(sb + kBwdSlotGo + off);
      const uint4 pj = *reinterpret_cast<const uint4 *>(sb + kBwdSlotProj + off);
      pc[c] = go_proj_chunk_dot(g, pj);
      // gos = bf16(go * inv_rms), as the reference's (grad_out * inv_rms).to(x.dtype)
      uint4 o;
      o.x = pack_bf16x2(bf16lo(g.x) * rinv, bf16hi(g.x) * rinv);
      o.y = pack_bf16x2(bf16lo(g.y) * rinv, bf16hi(g.y) * rinv);
      o.z = pack_bf16x2(bf16lo(g.z) * rinv, bf16hi(g.z) * rinv);
      o.w = pack_bf16x2(bf16lo(g.w) * rinv, bf16hi(g.w) * rinv);
      *reinterpret_cast<uint4 *>(sb + GOS + off) = o;
    }
    const float dot = (pc[0] + pc[1]) + (pc[2] + pc[3]);
    reinterpret_cast<float2 *>(sb + SINV)[r] =
        make_float2(dot * (rinv * rinv) / nC, rinv);
  }
}

__global__ void __launch_bounds__(kBwdThreads, 1)
k1_bwd_tc_kernel(const __grid_constant__ CUtensorMap tmap_x,
                 const __grid_constant__ CUtensorMap tmap_gx,
                 const __grid_constant__ CUtensorMap tmap_go,
                 const __grid_constant__ CUtensorMap tmap_proj,
                 const __grid_constant__ CUtensorMap tmap_w, const BwdArgs a) {
  extern __shared__ uint8_t smem_raw[];
  BwdSmem &sm = *reinterpret_cast<BwdSmem *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  volatile int *abort = &sm.abort;

  int grp, gi, ng;
  bwd_cta_group(int(blockIdx.x), a.base, a.rem, grp, gi, ng);
  const int G = a.G;
  const int ntiles = gi < a.ntt ? (a.ntt - gi + ng - 1) / ng : 0;
  const int nunits = ntiles * G;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kBwdStages; ++s) {
      mbar_init(smem_u32(&sm.full[s]), 1);
      mbar_init(smem_u32(&sm.empty[s]), 1);  // released by the store warp after its store read
      mbar_init(smem_u32(&sm.epi[s]), kBwdEpiWarps);
    }
    for (int b = 0; b < kBwdSlots; ++b) {
      mbar_init(smem_u32(&sm.gfull[b]), 1);
      mbar_init(smem_u32(&sm.gready[b]), 1);
      mbar_init(smem_u32(&sm.gempty[b]), 1 + kBwdEpiWarps);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&sm.tfull[b]), 1);
      mbar_init(smem_u32(&sm.tempty[b]), kBwdEpiWarps);
    }
    mbar_init(smem_u32(&sm.dwfull), 1);
    mbar_init(smem_u32(&sm.mma_done), 1);
    sm.abort = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_x);
    prefetch_tmap(&tmap_gx);
    prefetch_tmap(&tmap_go);
    prefetch_tmap(&tmap_proj);
    prefetch_tmap(&tmap_w);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&sm.tmem_base), kBwdTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  // No global memory is touched before this point (see pdl_wait()).
  pdl_wait();

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0, slot = 0, issued = 0, slots_issued = 0;
      uint32_t phase = 0, sphase = 0;
      const uint32_t gtx = uint32_t(2 * kBwdGBytes);
      for (int j = 0; j < nunits && !*abort; ++j) {
        const int m = j / G, jj = j - m * G;
        const int32_t row0 = (gi + m * ng) * kBwdBT;
        const int kc = grp * G + jj;
        if (jj == 0) {  // new token tile: go and proj into the next slot
          if (!mbar_wait(smem_u32(&sm.gempty[slot]), sphase ^ 1, abort, kSiteBProdSlot)) break;
          const uint32_t gf = smem_u32(&sm.gfull[slot]);
          const uint32_t sb = smem_u32(sm.slot[slot]);
          mbar_arrive_expect_tx(gf, gtx);
          tma_load_2d(sb + kBwdSlotGo, &tmap_go, gf, 0, row0);
          tma_load_2d(sb + kBwdSlotProj, &tmap_proj, gf, 0, row0);
          ++slots_issued;
          if (++slot == kBwdSlots) { slot = 0; sphase ^= 1; }
        }
        if (!mbar_wait(smem_u32(&sm.empty[stage]), phase ^ 1, abort, kSiteBProdEmpty)) break;
        const uint32_t f = smem_u32(&sm.full[stage]);
        const uint32_t base = smem_u32(sm.stage[stage]);
        mbar_arrive_expect_tx(f, uint32_t(kBwdStageBytes));
        tma_load_2d(base, &tmap_x, f, kc * kBwdBK, row0);
        tma_load_2d(base + kBwdXBox, &tmap_x, f, kc * kBwdBK + 64, row0);
        tma_load_2d(base + kBwdXBytes, &tmap_w, f, kc * kBwdBK, 0);
        tma_load_2d(base + kBwdXBytes + kBwdWBytes / 2, &tmap_w, f, kc * kBwdBK + 64, 0);
        ++issued;
        if (++stage == kBwdStages) { stage = 0; phase ^= 1; }
      }
      // Drain: every copy issued must have landed before the CTA exits.
      int n = issued < kBwdStages ? issued : kBwdStages;
      int s = stage;
      uint32_t ph = phase;
      for (int i = 0; i < n; ++i) {
        if (--s < 0) { s = kBwdStages - 1; ph ^= 1; }
        mbar_wait(smem_u32(&sm.full[s]), ph, abort, kSiteBDrain, true);
      }
      n = slots_issued < kBwdSlots ? slots_issued : kBwdSlots;
      s = slot;
      ph = sphase;
      for (int i = 0; i < n; ++i) {
        if (--s < 0) { s = kBwdSlots - 1; ph ^= 1; }
        mbar_wait(smem_u32(&sm.gfull[s]), ph, abort, kSiteBDrain, true);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc_dx = idesc_bf16_f32(kBwdBT, kBwdBK, 0, 1);
      constexpr uint32_t idesc_dw = idesc_bf16_f32(kBwdBK, kND, 1, 1);
      int stage = 0, acc = 0, slot = 0;
      uint32_t phase = 0, acc_phase = 0, sphase = 0;
      bool ok = true;
      for (int j = 0; j < nunits && !*abort; ++j) {
        const int m = j / G, jj = j - m * G;
        if (jj == 0 &&
            !mbar_wait(smem_u32(&sm.gready[slot]), sphase, abort, kSiteBMmaSlot)) { ok = false; break; }
        if (!mbar_wait(smem_u32(&sm.tempty[acc]), acc_phase ^ 1, abort, kSiteBMmaTempty)) { ok = false; break; }
        if (!mbar_wait(smem_u32(&sm.full[stage]), phase, abort, kSiteBMmaFull)) { ok = false; break; }
        tc_fence_after();
        const uint32_t base = smem_u32(sm.stage[stage]);
        const uint32_t gs = smem_u32(sm.slot[slot]);
        if (a.with_dw) {
          // grad_W: M = k (two 64-wide MN blocks 16 KiB apart), N = d, K = tokens.
#pragma unroll
          for (int k = 0; k < kBwdBT / 16; ++k) {
            const uint64_t ad = smem_desc(base + k * 2048, kBwdXBox, 1024, 2);
            const uint64_t bd = smem_desc(gs + kBwdSlotGos + k * 1024, 512, 512, 4);
            mma_bf16_ss(tmem + kBwdDwCol + uint32_t(jj * kND), ad, bd, idesc_dw,
                        (m > 0 || k > 0) ? 1u : 0u);
          }
        }
        {
          // grad_x: M = tokens, N = 128 k (two 64-wide MN blocks 4 KiB apart), K = d.
          const uint32_t wb = base + kBwdXBytes;
#pragma unroll
          for (int k = 0; k < kND / 16; ++k) {
            const uint64_t ad = smem_desc(gs + kBwdSlotGo + k * 32, 16, 512, 4);
            const uint64_t bd = smem_desc(wb + k * 2048, kBwdWBytes / 2, 1024, 2);
            mma_bf16_ss(tmem + uint32_t(acc * kBwdBK), ad, bd, idesc_dx, k != 0);
          }
        }
        mma_commit(smem_u32(&sm.tfull[acc]));
        if (jj == G - 1) {
          mma_commit(smem_u32(&sm.gempty[slot]));
          if (++slot == kBwdSlots) { slot = 0; sphase ^= 1; }
        }
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
        if (++stage == kBwdStages) { stage = 0; phase ^= 1; }
      }
      if (ok && !*abort && a.with_dw && nunits > 0) mma_commit(smem_u32(&sm.dwfull));
      mma_commit(smem_u32(&sm.mma_done));
      mbar_wait(smem_u32(&sm.mma_done), 0, abort, kSiteBDrain, true);
    }
  } else if (warp < kBwdStoreWarp) {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;           // TMEM lane quarter
    const int h = (warp - 2) >> 2;    // column half of the unit (0: 0-63, 1: 64-127)
    const int r = q * 32 + lane;      // token row of the unit / k row of the grad_W partial
    int stage = 0, acc = 0, slot = 0;
    uint32_t phase = 0, acc_phase = 0, sphase = 0;
    float s = 0.f, inv = 0.f;
    bool ok = true;
    for (int j = 0; j < nunits && !*abort; ++j) {
      const int m = j / G, jj = j - m * G;
      if (jj == 0) {
        // (s, inv_rms) of this thread's token, kept in registers for the tile.
        if (!mbar_wait(smem_u32(&sm.gready[slot]), sphase, abort, kSiteBEpiSlot)) { ok = false; break; }
        const float2 si = reinterpret_cast<const float2 *>(sm.slot[slot] + kBwdSlotSinv)[r];
        s = si.x;
        inv = si.y;
        // The slot's refill is a TMA (async-proxy) write: order this thread's
        // generic-proxy read before it, then release (one arrive per warp).
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.gempty[slot]));
        if (++slot == kBwdSlots) { slot = 0; sphase ^= 1; }
      }
      if (!mbar_wait(smem_u32(&sm.full[stage]), phase, abort, kSiteBEpiFull)) { ok = false; break; }
      uint8_t *xs = sm.stage[stage];
      if (!mbar_wait(smem_u32(&sm.tfull[acc]), acc_phase, abort, kSiteBEpiTfull)) { ok = false; break; }
      tc_fence_after();
      uint32_t v[2][32];
      const uint32_t tl = tmem + (uint32_t(q * 32) << 16) + uint32_t(acc * kBwdBK + 64 * h);
      tmem_ld_32x32b_x32(tl, v[0]);
      tmem_ld_32x32b_x32(tl + 32, v[1]);
      tmem_wait_ld();
      // Columns 64h .. 64h+63 of row r are one 128-byte row of x box h; read
      // all eight 16-byte chunks before the math so the loads overlap.
      uint8_t *rowp = xs + h * kBwdXBox + r * 128;
      uint4 xv[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) xv[i] = *reinterpret_cast<const uint4 *>(rowp + ((i ^ (r & 7)) << 4));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float *dv = reinterpret_cast<const float *>(v[i >> 2] + 8 * (i & 3));
        uint4 o;
        o.x = pack_bf16x2(fmaf(-s, bf16lo(xv[i].x), inv * dv[0]), fmaf(-s, bf16hi(xv[i].x), inv * dv[1]));
        o.y = pack_bf16x2(fmaf(-s, bf16lo(xv[i].y), inv * dv[2]), fmaf(-s, bf16hi(xv[i].y), inv * dv[3]));
        o.z = pack_bf16x2(fmaf(-s, bf16lo(xv[i].z), inv * dv[4]), fmaf(-s, bf16hi(xv[i].z), inv * dv[5]));
        o.w = pack_bf16x2(fmaf(-s, bf16lo(xv[i].w), inv * dv[6]), fmaf(-s, bf16hi(xv[i].w), inv * dv[7]));
        *reinterpret_cast<uint4 *>(rowp + ((i ^ (r & 7)) << 4)) = o;
      }
      // Every writer makes its grad_x visible to the TMA (async proxy), then
      // one arrive per warp on epi[stage] for the store warp and on tempty.
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_u32(&sm.epi[stage]));
        mbar_arrive(smem_u32(&sm.tempty[acc]));
      }
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      if (++stage == kBwdStages) { stage = 0; phase ^= 1; }
    }
    if (ok && a.with_dw && nunits > 0 &&
        mbar_wait(smem_u32(&sm.dwfull), 0, abort, kSiteBEpiDw)) {
      // grad_W partials of the group's G k-chunks: thread r owns k row r of
      // each, 32 d columns; warps 2-5 take the even chunks, warps 6-9 the odd.
      tc_fence_after();
      float *dst0 = a.dw_part + int64_t(blockIdx.x) * G * (kND * kBwdBK) + r;
      for (int jj = h; jj < G; jj += 2) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(tmem + (uint32_t(q * 32) << 16) + kBwdDwCol + uint32_t(jj * kND), v);
        tmem_wait_ld();
        float *dst = dst0 + int64_t(jj) * (kND * kBwdBK);
#pragma unroll
        for (int d = 0; d < kND; ++d) __stcg(dst + d * kBwdBK, __uint_as_float(v[d]));
      }
    }
  } else if (warp == kBwdStoreWarp) {
    // --------------------------------------------------------------- store
    if (lane == 0) {
      int stage = 0, npend = 0;
      int pend[kBwdInflight];
      uint32_t phase = 0;
      for (int j = 0; j < nunits && !*abort; ++j) {
        const int m = j / G, jj = j - m * G;
        const int32_t row0 = (gi + m * ng) * kBwdBT;
        const int kc = grp * G + jj;
        if (!mbar_wait(smem_u32(&sm.epi[stage]), phase, abort, kSiteBEpiStore)) break;
        const uint32_t base = smem_u32(sm.stage[stage]);
        tma_store_2d(&tmap_gx, base, kc * kBwdBK, row0);
        tma_store_2d(&tmap_gx, base + kBwdXBox, kc * kBwdBK + 64, row0);
        tma_store_commit();
        pend[npend++] = stage;
        // At most kBwdInflight - 1 older stores may still be reading shared
        // memory; the stages of all the others are free again.
        tma_store_wait_read<kBwdInflight - 1>();
        while (npend > kBwdInflight - 1) {
          mbar_arrive(smem_u32(&sm.empty[pend[0]]));
          for (int i = 1; i < npend; ++i) pend[i - 1] = pend[i];
          --npend;
        }
        if (++stage == kBwdStages) { stage = 0; phase ^= 1; }
      }
      tma_store_wait_all<0>();
      for (int i = 0; i < npend; ++i) mbar_arrive(smem_u32(&sm.empty[pend[i]]));
    }
  } else if (warp == kBwdPrepWarp) {
    // ----------------------------------------------------------- tile prep
    // Lane l takes the tile rows l, l + 32, l + 64, l + 96.  Rows of go, proj
    // and gos are 64 bytes with the TMA's 64-byte swizzle: 16-byte chunk c of
    // row r sits at chunk position c ^ ((r >> 1) & 3).
    int slot = 0;
    uint32_t sphase = 0;
    for (int m = 0; m < ntiles && !*abort; ++m) {
      const int64_t t0 = int64_t(gi + m * ng) * kBwdBT;
      float invr[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t t = t0 + lane + 32 * i;
        invr[i] = t < a.T ? __ldg(a.inv_rms + t) : 0.f;
      }
      if (!mbar_wait(smem_u32(&sm.gfull[slot]), sphase, abort, kSiteBPrepSlot)) break;
      prep_tile<kBwdSlotGos, kBwdSlotSinv>(sm.slot[slot], lane, invr, float(a.nC));
      // gos is read by the MMA (async proxy) and go/proj are refilled by the
      // TMA: order this thread's generic reads and writes before both.
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sm.gready[slot]));
      if (++slot == kBwdSlots) { slot = 0; sphase ^= 1; }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kBwdTmemCols);
  }
}

// grad_W[d, k] = bf16(sum of the grad_W partials of the CTAs of k's group),
// in increasing CTA order (deterministic).  Block (kc, d): row d of k-chunk
// kc, one thread per column.  The contributors are the group's CTAs that took
// at least one token tile (index i < ntt); their partials are loaded eight at
// a time and added in order.  (Four threads per column, each adding a quarter
// of the contributors, measured slower: 8.6 against 5.9 us.)
__global__ void __launch_bounds__(kBwdBK)
k1_bwd_dw_reduce_kernel(const float *__restrict__ part, __nv_bfloat16 *__restrict__ gW, int nC,
                        int ntt, int G, int base, int rem) {
  pdl_wait();
  const int kc = blockIdx.x, d = blockIdx.y, kl = threadIdx.x;
  const int g = kc / G, jj = kc - g * G;
  const int first = bwd_group_first_cta(g, base, rem);
  const int ng = g < rem ? base + 1 : base;
  const int n = ng < ntt ? ng : ntt;
  const int64_t stride = int64_t(G) * (kND * kBwdBK);
  const float *col = part + int64_t(first) * stride + (int64_t(jj) * kND + d) * kBwdBK + kl;
  float acc = 0.f;
  for (int i = 0; i < n; i += 8) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = (i + u < n) ? __ldg(col + int64_t(i + u) * stride) : 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u < n) acc += v[u];
  }
  // A CTA of the main kernel whose bounded wait gave up has not written its
  // partials, so the sum would mix in whatever the workspace held before.
  // While the device error word is set (until fmhc_check_device_error reads
  // and clears it) grad_W is therefore written as NaN, never as a plausible
  // value.  The main kernel completed before this grid passed pdl_wait(), so
  // its error store is visible here.
  if (*reinterpret_cast<volatile unsigned *>(&sm100::g_device_error) != 0u) acc = __int_as_float(0x7fc00000);
  gW[int64_t(d) * nC + int64_t(kc) * kBwdBK + kl] = __float2bfloat16_rn(acc);
}

}  // namespace k1tc
}  // namespace fmhc
