// K1 backward on the tensor cores from an 8-bit checkpoint of x: grad_x and
// grad_W in one pass over the codes.  Included by k1_tc.cu after
// k1_tc_bwd.cuh, whose formulas, work order, token-tile slots and grad_W
// reduction it shares (x there is the restored x8 here).
//
// The tensor cores want x as bf16 in the 128-byte-swizzled layout that the TMA
// gives the bf16 kernel.  Both code formats are exact in bf16, so eight more
// warps widen the codes into that layout:
//
//   warp 0       TMA producer: go and proj per token tile (slots), and per unit
//                the codes [128 t x 128 k] and the W chunk, each into a ring of
//                its own.
//   warps 12-19  converters, two warps per 32 token rows, thread = token row and
//                64 columns: codes and scale bytes -> bf16 x tile in a stage.
//                The four scale bytes of a row's 128 columns are one word,
//                loaded a unit ahead.
//   warp 1       MMA issuer, warps 2-9 epilogue, warp 10 store, warp 11 tile
//                prep: as in the bf16 kernel; the epilogue takes its 64 columns
//                in two halves, which keeps a thread within the 96 registers
//                that 20 warps leave, and the prep writes gos over proj.
//
// Codes are free again once converted, W once the MMAs of its unit are done, a
// stage once the store has read the grad_x that the epilogue wrote over x.
//
// What bounds it: shared memory.  A unit moves 48 KiB of HBM traffic but about
// 220 KiB through shared memory (codes in and out, x in, to the MMAs and to the
// epilogue, grad_x in and out), on top of the 64 KiB of HBM and 180 KiB of the
// bf16 kernel.  T = 65536, C = 1024, int8, us (bf16 kernel: 181; floor of the
// bytes: 126): four converter warps 216; eight 189; codes and W in rings of
// their own 182; codes ahead of W and one store held 174; rings of 4 codes, 4 W,
// 3 stages instead of 3, 2, 4: 166.  Not faster: codes loaded into registers
// (241), converter and epilogue in one warp with x kept in registers (171), the
// same with D1 a unit ahead and grad_x in tiles of its own (193), codes of two
// chunks at a time (175), a slot loaded half a tile ahead (172), the epilogue's
// two halves on alternate units (178: a stage is held longer).
// Every wait is bounded (sm100_ptx.cuh).
#pragma once

#include "act8.cuh"
#include "lane_ring.cuh"

namespace fmhc {
namespace k1tc {

constexpr int kQ8Codes = 4;                   // code tiles in flight
constexpr int kQ8W = 4;                       // W chunks in flight
constexpr int kQ8Stages = 3;                  // x tiles
constexpr int kQ8CodeBytes = kBwdBT * kBwdBK;  // 16 KiB
constexpr int kQ8ConvWarp = kBwdPrepWarp + 1;
constexpr int kQ8ConvWarps = 8;
constexpr int kQ8Threads = 32 * (kQ8ConvWarp + kQ8ConvWarps);  // 640
// Slot layout: go at 0, proj and later gos at 8 KiB, (s, inv) at 16 KiB.
constexpr int kQ8SlotGos = kBwdSlotProj, kQ8SlotSinv = 2 * kBwdGBytes;
constexpr int kQ8SlotBytes = 2 * kBwdGBytes + kBwdSBytes;

struct alignas(1024) BwdQ8Smem {
  uint8_t x[kQ8Stages][kBwdXBytes];           // x tile, later grad_x
  uint8_t codes[kQ8Codes][kQ8CodeBytes];
  uint8_t w[kQ8W][kBwdWBytes];
  uint8_t slot[kBwdSlots][kQ8SlotBytes];      // go, proj or gos, (s, inv) of one token tile
  uint64_t cfull[kQ8Codes];                   // codes landed
  uint64_t cempty[kQ8Codes];                  // converters have read them
  uint64_t wfull[kQ8W];                       // W landed
  uint64_t wempty[kQ8W];                      // the MMAs have read it
  uint64_t xfull[kQ8Stages];                  // converters wrote x
  uint64_t empty[kQ8Stages];                  // the store has read grad_x
  uint64_t epi[kQ8Stages];                    // the epilogue wrote grad_x
  uint64_t gfull[kBwdSlots];
  uint64_t gready[kBwdSlots];
  uint64_t gempty[kBwdSlots];
  uint64_t tfull[2];
  uint64_t tempty[2];
  uint64_t dwfull;
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort;
};

enum : unsigned { kSiteQProdCodes = 0x301, kSiteQProdSlot = 0x302, kSiteQMmaW = 0x303,
                  kSiteQMmaX = 0x304, kSiteQMmaTempty = 0x305, kSiteQMmaSlot = 0x306,
                  kSiteQEpiSlot = 0x307, kSiteQEpiX = 0x308, kSiteQEpiTfull = 0x309,
                  kSiteQEpiDw = 0x30a, kSiteQStore = 0x30b, kSiteQPrep = 0x30c,
                  kSiteQConvX = 0x30d, kSiteQConvCodes = 0x30e, kSiteQProdW = 0x30f,
                  kSiteQDrain = 0x310 };

// mbar_wait by a whole warp with one outcome: a lane whose wait expires takes the
// others with it, so that no lane is left at a warp barrier.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int *abort,
                                               unsigned site) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, site));
}

template <int FMT>
__global__ void __launch_bounds__(kQ8Threads, 1)
k1_bwd_q8_tc_kernel(const __grid_constant__ CUtensorMap tmap_codes,
                    const __grid_constant__ CUtensorMap tmap_gx,
                    const __grid_constant__ CUtensorMap tmap_go,
                    const __grid_constant__ CUtensorMap tmap_proj,
                    const __grid_constant__ CUtensorMap tmap_w,
                    const uint8_t *__restrict__ scales, const BwdArgs a) {
  // No static shared memory beside it, so it starts on a 1 KiB boundary.
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  BwdQ8Smem &sm = *reinterpret_cast<BwdQ8Smem *>(smem_raw);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  volatile int *abort = &sm.abort;

  int grp, gi, ng;
  bwd_cta_group(int(blockIdx.x), a.base, a.rem, grp, gi, ng);
  const int G = a.G;
  const int ntiles = gi < a.ntt ? (a.ntt - gi + ng - 1) / ng : 0;
  const int nunits = ntiles * G;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kQ8Codes; ++s) {
      mbar_init(smem_u32(&sm.cfull[s]), 1);
      mbar_init(smem_u32(&sm.cempty[s]), kQ8ConvWarps);
    }
    for (int s = 0; s < kQ8W; ++s) {
      mbar_init(smem_u32(&sm.wfull[s]), 1);
      mbar_init(smem_u32(&sm.wempty[s]), 1);
    }
    for (int s = 0; s < kQ8Stages; ++s) {
      mbar_init(smem_u32(&sm.xfull[s]), kQ8ConvWarps);
      mbar_init(smem_u32(&sm.empty[s]), 1);
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
    prefetch_tmap(&tmap_codes);
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
      int cs = 0, ws = 0, slot = 0, issued = 0, w_issued = 0, slots_issued = 0;
      uint32_t cphase = 0, wphase = 0, sphase = 0;
      // Unit j's codes go out before unit j - 1's W chunk: waiting for the MMAs
      // to release a W chunk must not hold back the codes.
      for (int j = 0; j <= nunits && !*abort; ++j) {
        const int m = j / G, jj = j - m * G;
        const int32_t row0 = (gi + m * ng) * kBwdBT;
        const int kc = grp * G + jj;
        if (j < nunits) {
          if (jj == 0) {  // new token tile: go and proj into the next slot
            if (!mbar_wait(smem_u32(&sm.gempty[slot]), sphase ^ 1, abort, kSiteQProdSlot)) break;
            const uint32_t gf = smem_u32(&sm.gfull[slot]);
            const uint32_t sb = smem_u32(sm.slot[slot]);
            mbar_arrive_expect_tx(gf, uint32_t(2 * kBwdGBytes));
            tma_load_2d(sb + kBwdSlotGo, &tmap_go, gf, 0, row0);
            tma_load_2d(sb + kBwdSlotProj, &tmap_proj, gf, 0, row0);
            ++slots_issued;
            if (++slot == kBwdSlots) { slot = 0; sphase ^= 1; }
          }
          if (!mbar_wait(smem_u32(&sm.cempty[cs]), cphase ^ 1, abort, kSiteQProdCodes)) break;
          const uint32_t cf = smem_u32(&sm.cfull[cs]);
          mbar_arrive_expect_tx(cf, uint32_t(kQ8CodeBytes));
          // The codes' map counts pairs of bytes: 64 of them are 128 columns.
          tma_load_2d(smem_u32(sm.codes[cs]), &tmap_codes, cf, kc * (kBwdBK / 2), row0);
          ++issued;
          if (++cs == kQ8Codes) { cs = 0; cphase ^= 1; }
        }
        if (j > 0) {
          const int kw = grp * G + (j - 1) % G;
          if (!mbar_wait(smem_u32(&sm.wempty[ws]), wphase ^ 1, abort, kSiteQProdW)) break;
          const uint32_t wf = smem_u32(&sm.wfull[ws]);
          mbar_arrive_expect_tx(wf, uint32_t(kBwdWBytes));
          tma_load_2d(smem_u32(sm.w[ws]), &tmap_w, wf, kw * kBwdBK, 0);
          tma_load_2d(smem_u32(sm.w[ws]) + kBwdWBytes / 2, &tmap_w, wf, kw * kBwdBK + 64, 0);
          ++w_issued;
          if (++ws == kQ8W) { ws = 0; wphase ^= 1; }
        }
      }
      // Drain: every copy issued must have landed before the CTA exits.
      int n = issued < kQ8Codes ? issued : kQ8Codes;
      int s = cs;
      uint32_t ph = cphase;
      for (int i = 0; i < n; ++i) {
        if (--s < 0) { s = kQ8Codes - 1; ph ^= 1; }
        mbar_wait(smem_u32(&sm.cfull[s]), ph, abort, kSiteQDrain, true);
      }
      n = w_issued < kQ8W ? w_issued : kQ8W;
      s = ws;
      ph = wphase;
      for (int i = 0; i < n; ++i) {
        if (--s < 0) { s = kQ8W - 1; ph ^= 1; }
        mbar_wait(smem_u32(&sm.wfull[s]), ph, abort, kSiteQDrain, true);
      }
      n = slots_issued < kBwdSlots ? slots_issued : kBwdSlots;
      s = slot;
      ph = sphase;
      for (int i = 0; i < n; ++i) {
        if (--s < 0) { s = kBwdSlots - 1; ph ^= 1; }
        mbar_wait(smem_u32(&sm.gfull[s]), ph, abort, kSiteQDrain, true);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc_dx = idesc_bf16_f32(kBwdBT, kBwdBK, 0, 1);
      constexpr uint32_t idesc_dw = idesc_bf16_f32(kBwdBK, kND, 1, 1);
      int stage = 0, ws = 0, acc = 0, slot = 0;
      uint32_t phase = 0, wphase = 0, acc_phase = 0, sphase = 0;
      bool ok = true;
      for (int j = 0; j < nunits && !*abort; ++j) {
        const int m = j / G, jj = j - m * G;
        if (jj == 0 &&
            !mbar_wait(smem_u32(&sm.gready[slot]), sphase, abort, kSiteQMmaSlot)) { ok = false; break; }
        if (!mbar_wait(smem_u32(&sm.tempty[acc]), acc_phase ^ 1, abort, kSiteQMmaTempty)) { ok = false; break; }
        if (!mbar_wait(smem_u32(&sm.wfull[ws]), wphase, abort, kSiteQMmaW)) { ok = false; break; }
        if (!mbar_wait(smem_u32(&sm.xfull[stage]), phase, abort, kSiteQMmaX)) { ok = false; break; }
        tc_fence_after();
        const uint32_t base = smem_u32(sm.x[stage]);
        const uint32_t wb = smem_u32(sm.w[ws]);
        const uint32_t gs = smem_u32(sm.slot[slot]);
        // grad_W: M = k (two 64-wide MN blocks 16 KiB apart), N = d, K = tokens.
#pragma unroll
        for (int k = 0; k < kBwdBT / 16; ++k) {
          const uint64_t ad = smem_desc(base + k * 2048, kBwdXBox, 1024, 2);
          const uint64_t bd = smem_desc(gs + kQ8SlotGos + k * 1024, 512, 512, 4);
          mma_bf16_ss(tmem + kBwdDwCol + uint32_t(jj * kND), ad, bd, idesc_dw,
                      (m > 0 || k > 0) ? 1u : 0u);
        }
        // grad_x: M = tokens, N = 128 k (two 64-wide MN blocks 4 KiB apart), K = d.
#pragma unroll
        for (int k = 0; k < kND / 16; ++k) {
          const uint64_t ad = smem_desc(gs + kBwdSlotGo + k * 32, 16, 512, 4);
          const uint64_t bd = smem_desc(wb + k * 2048, kBwdWBytes / 2, 1024, 2);
          mma_bf16_ss(tmem + uint32_t(acc * kBwdBK), ad, bd, idesc_dx, k != 0);
        }
        mma_commit(smem_u32(&sm.tfull[acc]));
        mma_commit(smem_u32(&sm.wempty[ws]));
        if (++ws == kQ8W) { ws = 0; wphase ^= 1; }
        if (jj == G - 1) {
          mma_commit(smem_u32(&sm.gempty[slot]));
          if (++slot == kBwdSlots) { slot = 0; sphase ^= 1; }
        }
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
        if (++stage == kQ8Stages) { stage = 0; phase ^= 1; }
      }
      if (ok && !*abort && nunits > 0) mma_commit(smem_u32(&sm.dwfull));
      mma_commit(smem_u32(&sm.mma_done));
      mbar_wait(smem_u32(&sm.mma_done), 0, abort, kSiteQDrain, true);
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
        if (!mbar_wait_warp(smem_u32(&sm.gready[slot]), sphase, abort, kSiteQEpiSlot)) { ok = false; break; }
        const float2 si = reinterpret_cast<const float2 *>(sm.slot[slot] + kQ8SlotSinv)[r];
        s = si.x;
        inv = si.y;
        // The slot's refill is a TMA (async-proxy) write: order this thread's
        // generic-proxy read before it, then release (one arrive per warp).
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.gempty[slot]));
        if (++slot == kBwdSlots) { slot = 0; sphase ^= 1; }
      }
      if (!mbar_wait_warp(smem_u32(&sm.xfull[stage]), phase, abort, kSiteQEpiX)) { ok = false; break; }
      if (!mbar_wait_warp(smem_u32(&sm.tfull[acc]), acc_phase, abort, kSiteQEpiTfull)) { ok = false; break; }
      tc_fence_after();
      // Columns 64h .. 64h+63 of row r are one 128-byte row of x box h.
      uint8_t *rowp = sm.x[stage] + h * kBwdXBox + r * 128;
      const uint32_t tl = tmem + (uint32_t(q * 32) << 16) + uint32_t(acc * kBwdBK + 64 * h);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(tl + 32 * p, v);
        uint4 xv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          xv[i] = *reinterpret_cast<const uint4 *>(rowp + (((4 * p + i) ^ (r & 7)) << 4));
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float *dv = reinterpret_cast<const float *>(v + 8 * i);
          uint4 o;
          o.x = pack_bf16x2(fmaf(-s, bf16lo(xv[i].x), inv * dv[0]), fmaf(-s, bf16hi(xv[i].x), inv * dv[1]));
          o.y = pack_bf16x2(fmaf(-s, bf16lo(xv[i].y), inv * dv[2]), fmaf(-s, bf16hi(xv[i].y), inv * dv[3]));
          o.z = pack_bf16x2(fmaf(-s, bf16lo(xv[i].z), inv * dv[4]), fmaf(-s, bf16hi(xv[i].z), inv * dv[5]));
          o.w = pack_bf16x2(fmaf(-s, bf16lo(xv[i].w), inv * dv[6]), fmaf(-s, bf16hi(xv[i].w), inv * dv[7]));
          *reinterpret_cast<uint4 *>(rowp + (((4 * p + i) ^ (r & 7)) << 4)) = o;
        }
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
      if (++stage == kQ8Stages) { stage = 0; phase ^= 1; }
    }
    if (ok && nunits > 0 && mbar_wait_warp(smem_u32(&sm.dwfull), 0, abort, kSiteQEpiDw)) {
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
      int stage = 0;
      uint32_t phase = 0;
      for (int j = 0; j < nunits && !*abort; ++j) {
        const int m = j / G, jj = j - m * G;
        const int32_t row0 = (gi + m * ng) * kBwdBT;
        const int kc = grp * G + jj;
        if (!mbar_wait(smem_u32(&sm.epi[stage]), phase, abort, kSiteQStore)) break;
        const uint32_t base = smem_u32(sm.x[stage]);
        tma_store_2d(&tmap_gx, base, kc * kBwdBK, row0);
        tma_store_2d(&tmap_gx, base + kBwdXBox, kc * kBwdBK + 64, row0);
        tma_store_commit();
        // Free the stage as soon as this store has read it (holding it until
        // the next store is issued, as the bf16 kernel does: 176 against 174 us).
        tma_store_wait_read<0>();
        mbar_arrive(smem_u32(&sm.empty[stage]));
        if (++stage == kQ8Stages) { stage = 0; phase ^= 1; }
      }
      tma_store_wait_all<0>();
    }
  } else if (warp == kBwdPrepWarp) {
    // ----------------------------------------------------------- tile prep
    // As in the bf16 kernel: lane l takes the tile rows l, l + 32, l + 64, l + 96.
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
      if (!mbar_wait_warp(smem_u32(&sm.gfull[slot]), sphase, abort, kSiteQPrep)) break;
      prep_tile<kQ8SlotGos, kQ8SlotSinv>(sm.slot[slot], lane, invr, float(a.nC));
      // gos is read by the MMA (async proxy) and go/proj are refilled by the
      // TMA: order this thread's generic reads and writes before both.
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sm.gready[slot]));
      if (++slot == kBwdSlots) { slot = 0; sphase ^= 1; }
    }
  } else {
    // ----------------------------------------------------------- converters
    const int r = ((warp - kQ8ConvWarp) & 3) * 32 + lane;  // token row of the unit
    const int h = (warp - kQ8ConvWarp) >> 2;               // x box: columns 64h .. 64h+63
    // Scale bytes 2h and 2h + 1 of the row's 128 columns (even addresses: nC / 32
    // is a multiple of 4, and the base is checked).
    const auto scale_pair = [&](int j) {
      const int m = j / G, kc = grp * G + (j - m * G);
      const int64_t t = int64_t(gi + m * ng) * kBwdBT + r;
      return j < nunits && t < a.T
                 ? uint32_t(__ldg(reinterpret_cast<const uint16_t *>(
                       scales + t * (a.nC / act8::kBlock) + kc * (kBwdBK / act8::kBlock) + 2 * h)))
                 : 0u;
    };
    int cs = 0, stage = 0;
    uint32_t cphase = 0, phase = 0;
    uint32_t next = scale_pair(0);
    for (int j = 0; j < nunits && !*abort; ++j) {
      const uint32_t sw = next;
      next = scale_pair(j + 1);
      if (!mbar_wait_warp(smem_u32(&sm.cfull[cs]), cphase, abort, kSiteQConvCodes)) break;
      // Row r of the codes: 128 bytes, 16-byte chunk c at position c ^ (r & 7);
      // chunks 4h .. 4h+3 are this thread's.  Chunk 4h + i goes to chunks 2i and
      // 2i + 1 of the 128-byte row r of x box h, swizzled the same way.
      const uint8_t *src = sm.codes[cs] + r * 128;
      uint4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint4 *>(src + (((4 * h + i) ^ (r & 7)) << 4));
      const uint32_t f0 = act8::widen_factor<FMT>(sw & 0xffu), f1 = act8::widen_factor<FMT>(sw >> 8);
      if (!mbar_wait_warp(smem_u32(&sm.empty[stage]), phase ^ 1, abort, kSiteQConvX)) break;
      uint8_t *row = sm.x[stage] + h * kBwdXBox + r * 128;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t f = i < 2 ? f0 : f1;
        const uint2 a0 = act8::widen4<FMT>(v[i].x, f), a1 = act8::widen4<FMT>(v[i].y, f);
        const uint2 b0 = act8::widen4<FMT>(v[i].z, f), b1 = act8::widen4<FMT>(v[i].w, f);
        *reinterpret_cast<uint4 *>(row + (((2 * i) ^ (r & 7)) << 4)) = make_uint4(a0.x, a0.y, a1.x, a1.y);
        *reinterpret_cast<uint4 *>(row + (((2 * i + 1) ^ (r & 7)) << 4)) = make_uint4(b0.x, b0.y, b1.x, b1.y);
      }
      // x is read by the MMA (async proxy) and the codes' place is refilled by
      // the TMA: order this thread's writes and reads before both.
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_u32(&sm.xfull[stage]));
        mbar_arrive(smem_u32(&sm.cempty[cs]));
      }
      if (++cs == kQ8Codes) { cs = 0; cphase ^= 1; }
      if (++stage == kQ8Stages) { stage = 0; phase ^= 1; }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kBwdTmemCols);
  }
}

}  // namespace k1tc
}  // namespace fmhc
