// K1 backward from an 8-bit checkpoint of x for little work, and for the widths
// that the tcgen05 kernel (k1_tc_bwd_q8.cuh) does not take: C % 32 != 0, where
// blocks of 32 do not line up with its tiles and rows of 4 C codes need not be what
// the TMA wants, and widths without a work split (k1_bwd_plan.h).
//
//   s       = (go . proj) inv^2 / nC
//   grad_x  = bf16( inv (go W) - s x8 )
//   grad_W  = bf16( sum over tokens of bf16(go inv)^T x8 )
//
// A block takes 256 of the nC columns and every gridDim.y-th tile of 32 tokens,
// through a shared-memory ring; a warp its own 32 columns of them: it widens
// their codes into a bf16 tile, feeds both products' warp-wide MMAs (m16n8k16)
// from it, writes grad_x over x8 and stores it.  Its columns of W stay in
// registers as MMA operands, its share of grad_W as accumulators.  Blocks of one
// column range (their tokens differ) write partials of grad_W, which
// k1_dw_sum_kernel adds in order; a single one writes grad_W itself.
//
// What bounds it: instructions, 20 or so per code, at two blocks of 128 registers
// per SM (three of 80 are slower, 437 against 330 us).  T = 65536, C = 1000, int8,
// us (floor of the bytes 121): codes loaded into registers a tile at a time, tiles
// of 64 tokens 428, of 32 394; scale bytes, go and proj through the ring too, and
// no bank conflicts 334; fewer instructions around the MMAs 330.  C = 1023, T =
// 3000: 30 (restoring x and the bf16 kernel for any width: 506).
#include "act8.cuh"
#include "fmhc_launch.h"
#include "grid.cuh"
#include "lane_ring.cuh"

#include <algorithm>

namespace fmhc {

using namespace act8;
using bf16 = __nv_bfloat16;

namespace {

constexpr int kD = 32;                  // projection width
constexpr int kTok = 32;                // tokens per tile
constexpr int kCols = 256, kWarps = 8;  // columns per block, 32 per warp
constexpr int kThreads = 32 * kWarps;
constexpr int kStages = 4;              // ring depth in tiles
constexpr int kBlocksPerSm = 2;
constexpr int kLoads = kTok / 4;        // of four codes each, per lane and tile
constexpr int kGPitch = kD + 8;         // bf16: an odd multiple of 16 bytes (ldmatrix)
// A row's scale bytes for the block's columns, in words: 11 bytes from the first word
// on hold them for every width and column range (tried for all C up to 2200).
constexpr int kScaleWords = 3;

struct AnySmem {
  uint8_t codes[kWarps][kStages][kTok][32];
  bf16 x[kWarps][kTok][32];           // x8, later grad_x; see x_at
  bf16 go[kStages][kTok][kGPitch];
  bf16 proj[kStages][kTok][kD];
  float inv[kStages][kTok];
  uint32_t scales[kStages][kTok][kScaleWords];
  bf16 gos[kTok][kGPitch];            // bf16(go inv)
  float2 sinv[kTok];
};
// Row r, column c (a multiple of 2) of a warp's x tile.  Two 64-byte rows make a
// line of all banks; the 16-byte chunks of a row are permuted by its line, so that
// eight rows' chunks (ldmatrix), a row's neighbouring columns and the MMA's
// accumulator places are all free of conflicts.
__device__ __forceinline__ bf16 *x_at(bf16 (*x)[32], int r, int c) {
  return &x[r][(((c >> 3) ^ ((r >> 1) & 3)) << 3) + (c & 7)];
}

__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], const bf16 *p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(uint32_t(__cvta_generic_to_shared(p)))
               : "memory");
}
__device__ __forceinline__ void load_matrices_t(uint32_t (&r)[4], const bf16 *p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(uint32_t(__cvta_generic_to_shared(p)))
               : "memory");
}
// d += a b
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// d = a b
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// To shared memory, `valid` bytes of BYTES from global memory and zeros.
template <int BYTES>
__device__ __forceinline__ void copy_or_zero(void *dst, const void *src, int valid) {
  static_assert(BYTES == 16 || BYTES == 4, "copy size");
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared_addr(dst)), "l"(src), "r"(valid)
                 : "memory");
  else
    copy_async4(shared_addr(dst), src, valid);
}

// WORD (C % 4 == 0): four neighbouring codes of a row are in one block.
template <int FMT, bool WORD>
__global__ void __launch_bounds__(32 * kWarps, kBlocksPerSm)
k1_bwd_q8_any_kernel(const bf16 *__restrict__ go, const uint8_t *__restrict__ codes,
                     const uint8_t *__restrict__ scales, const bf16 *__restrict__ W,
                     const bf16 *__restrict__ proj, const float *__restrict__ inv_rms,
                     bf16 *__restrict__ gx, bf16 *__restrict__ gW, float *__restrict__ part,
                     int64_t T, int nC, int64_t tiles) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  AnySmem &sm = *reinterpret_cast<AnySmem *>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int C = nC / 4, nb = (C + kBlock - 1) / kBlock;
  const int k0 = blockIdx.x * kCols, kw = k0 + warp * 32;  // the block's and the warp's first column
  const bool active = kw < nC;                             // uniform in the warp
  // Codes and grad_x: eight lanes hold the 32 columns of a row, four each.
  const int row8 = lane >> 3, c4 = (lane & 7) * 4, col = kw + c4;
  const bool in_col = col < nC;  // nC is a multiple of 4
  // Scale bytes lie in a row of 4 nb (whole words) at block_of(column).
  const auto block_of = [&](int k) { return k / C * nb + k % C / kBlock; };
  const int first_word = block_of(k0) / 4, row_words = nb;
  int s_off[WORD ? 1 : 4];  // of the lane's codes, from the first word on
#pragma unroll
  for (int i = 0; i < (WORD ? 1 : 4); ++i) s_off[i] = in_col ? block_of(col + i) - 4 * first_word : 0;
  pdl_wait();
  // W as the second operand of go W: [n tile][k step][half of the step's 16 d].
  uint32_t wf[4][2][2];
#pragma unroll
  for (int nt = 0; nt < 4; ++nt)
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = kw + nt * 8 + (lane >> 2), d = ks * 16 + h * 8 + (lane & 3) * 2;
        uint32_t lo = 0, hi = 0;
        if (k < nC) {
          lo = __ldg(reinterpret_cast<const uint16_t *>(W) + int64_t(d) * nC + k);
          hi = __ldg(reinterpret_cast<const uint16_t *>(W) + int64_t(d + 1) * nC + k);
        }
        wf[nt][ks][h] = lo | hi << 16;
      }
  float dw[2][4][4];  // grad_W: [16 d][n tile]
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int nt = 0; nt < 4; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) dw[i][nt][k] = 0.f;
  const int mi = lane >> 3, mr = lane & 7;  // ldmatrix: matrix and row whose address a lane gives
  bf16(*const x)[32] = sm.x[warp];
  // Tile m into a stage, zeros past the last token and column.  Codes: rows of a
  // multiple of 16 bytes (WORD) in copies of 16, others of 4.
  const auto fetch = [&](int64_t m, int stage) {
    if (m < tiles) {
      const int64_t t0 = m * kTok;
      const int left = int(min(T - t0, int64_t(kTok)));
      if (active) {
        constexpr int B = WORD ? 16 : 4, kPerRow = 32 / B, kRows = 32 / kPerRow;
        const int r = lane / kPerRow, c = lane % kPerRow * B;
        const uint8_t *src = codes + (t0 + r) * nC + kw + c;
#pragma unroll
        for (int i = 0; i < kTok; i += kRows) {
          const bool in = kw + c < nC && r + i < left;
          copy_or_zero<B>(&sm.codes[warp][stage][r + i][c], in ? src + i * int64_t(nC) : codes, in ? B : 0);
        }
      }
      {  // eight threads per token: 16 bytes of go or proj each
        static_assert(kThreads == 8 * kTok, "a thread per copy");
        const int r = threadIdx.x >> 3, c = (threadIdx.x & 3) * 8;
        const bool in = r < left, is_go = (threadIdx.x & 4) == 0;
        copy_or_zero<16>(is_go ? &sm.go[stage][r][c] : &sm.proj[stage][r][c],
                         (is_go ? go : proj) + (in ? (t0 + r) * kD + c : 0), in ? 16 : 0);
      }
      if (threadIdx.x < kTok * kScaleWords) {
        const int r = threadIdx.x / kScaleWords, w = threadIdx.x % kScaleWords;
        const bool in = r < left && first_word + w < row_words;
        copy_or_zero<4>(&sm.scales[stage][r][w],
                        scales + (in ? ((t0 + r) * row_words + first_word + w) * 4 : 0), in ? 4 : 0);
      } else if (threadIdx.x < kTok * (kScaleWords + 1)) {
        const int r = threadIdx.x - kTok * kScaleWords;
        const bool in = r < left;
        copy_or_zero<4>(&sm.inv[stage][r], inv_rms + (in ? t0 + r : 0), in ? 4 : 0);
      }
    }
    copy_commit();
  };
  const int64_t step = gridDim.y;
  int64_t m = blockIdx.y;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) fetch(m + s * step, s);
  int stage = 0;
  for (; m < tiles; m += step) {
    const int64_t t0 = m * kTok;
    const int left = int(min(T - t0, int64_t(kTok)));  // tokens of this tile
    copy_wait<kStages - 2>();
    __syncthreads();  // the stage is there, and the one before it read by all
    fetch(m + (kStages - 1) * step, stage == 0 ? kStages - 1 : stage - 1);
    {  // bf16(go inv) and s: eight threads per token, four of the 32 d each
      const int r = threadIdx.x >> 3, d = (threadIdx.x & 7) * 4;
      const uint2 g = *reinterpret_cast<const uint2 *>(&sm.go[stage][r][d]);
      const uint2 p = *reinterpret_cast<const uint2 *>(&sm.proj[stage][r][d]);
      const float inv = sm.inv[stage][r];
      float dot = bf16lo(g.x) * bf16lo(p.x);
      dot = fmaf(bf16hi(g.x), bf16hi(p.x), dot);
      dot = fmaf(bf16lo(g.y), bf16lo(p.y), dot);
      dot = fmaf(bf16hi(g.y), bf16hi(p.y), dot);
#pragma unroll
      for (int o = 1; o < 8; o *= 2) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      *reinterpret_cast<uint2 *>(&sm.gos[r][d]) =
          make_uint2(pack_bf16x2(bf16lo(g.x) * inv, bf16hi(g.x) * inv),
                     pack_bf16x2(bf16lo(g.y) * inv, bf16hi(g.y) * inv));
      if (d == 0) sm.sinv[r] = make_float2(dot * (inv * inv) / float(nC), inv);
    }
    if (active) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int r = i * 4 + row8;
        const uint32_t w = *reinterpret_cast<const uint32_t *>(&sm.codes[warp][stage][r][c4]);
        const uint8_t *s = reinterpret_cast<const uint8_t *>(sm.scales[stage][r]);
        uint2 v;
        if constexpr (WORD) {
          v = widen4<FMT>(w, widen_factor<FMT>(s[s_off[0]]));
        } else {
          float f[4];
          decode4<FMT>(w, f);
#pragma unroll
          for (int k = 0; k < 4; ++k) f[k] *= scale_value(s[s_off[k]]);
          v = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
        }
        *reinterpret_cast<uint2 *>(x_at(x, r, c4)) = v;
      }
    }
    __syncthreads();  // gos and s, and the warp's x8
    if (active) {
      // grad_W += gos^T x8: first operand d x tokens, second tokens x columns,
      // both from rows of tokens.
#pragma unroll
      for (int ks = 0; ks < kTok / 16; ++ks) {
        uint32_t a[2][4], b[4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
          load_matrices_t(a[i], &sm.gos[ks * 16 + (mi >> 1) * 8 + mr][i * 16 + (mi & 1) * 8]);
#pragma unroll
        for (int np = 0; np < 2; ++np) {
          load_matrices_t(b, x_at(x, ks * 16 + (mi & 1) * 8 + mr, np * 16 + (mi >> 1) * 8));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            mma(dw[i][2 * np], a[i], b[0], b[1]);
            mma(dw[i][2 * np + 1], a[i], b[2], b[3]);
          }
        }
      }
      __syncwarp();  // x8 is overwritten below
#pragma unroll
      for (int mt = 0; mt < kTok / 16; ++mt) {
        float acc[4][4];
        uint32_t a[2][4];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
          load_matrices(a[ks], &sm.go[stage][mt * 16 + (mi & 1) * 8 + mr][ks * 16 + (mi >> 1) * 8]);
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) mma_first(acc[nt], a[0], wf[nt][0][0], wf[nt][0][1]);
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) mma(acc[nt], a[1], wf[nt][1][0], wf[nt][1][1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = mt * 16 + h * 8 + (lane >> 2);
          const float2 si = sm.sinv[r];
#pragma unroll
          for (int nt = 0; nt < 4; ++nt) {
            uint32_t *p = reinterpret_cast<uint32_t *>(x_at(x, r, nt * 8 + (lane & 3) * 2));
            const uint32_t v = *p;
            const float2 g = mul2(both(si.y), make_float2(acc[nt][2 * h], acc[nt][2 * h + 1]));
            const float2 o = fma2(both(-si.x), make_float2(bf16lo(v), bf16hi(v)), g);
            *p = pack_bf16x2(o.x, o.y);
          }
        }
      }
      __syncwarp();
      bf16 *dst = gx + (t0 + row8) * nC + col;
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        if (in_col && i * 4 + row8 < left)
          __stcs(reinterpret_cast<uint2 *>(dst + i * 4 * int64_t(nC)),
                 *reinterpret_cast<const uint2 *>(x_at(x, i * 4 + row8, c4)));
      __syncwarp();  // the next tile's x8 goes to the same place
    }
    if (++stage == kStages) stage = 0;
  }
  if (!active) return;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int nt = 0; nt < 4; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int d = i * 16 + h * 8 + (lane >> 2), k = kw + nt * 8 + (lane & 3) * 2;
        if (k >= nC) continue;  // nC is even
        const float a = dw[i][nt][2 * h], b = dw[i][nt][2 * h + 1];
        if (gridDim.y == 1) {
          gW[int64_t(d) * nC + k] = __float2bfloat16_rn(a);
          gW[int64_t(d) * nC + k + 1] = __float2bfloat16_rn(b);
        } else {
          *reinterpret_cast<float2 *>(part + (int64_t(blockIdx.y) * kD + d) * nC + k) = make_float2(a, b);
        }
      }
}

// grad_W from n partials, in a fixed order: a block takes 32 sums, each of its
// warps every eighth partial.
constexpr int kSumWarps = 8;
__global__ void __launch_bounds__(32 * kSumWarps)
k1_dw_sum_kernel(const float *__restrict__ part, bf16 *__restrict__ gW, int n, int64_t len) {
  __shared__ float acc[kSumWarps][32];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t j = int64_t(blockIdx.x) * 32 + lane;  // len is a multiple of 32
  float a = 0.f;
#pragma unroll 8
  for (int i = warp; i < n; i += kSumWarps) a += part[i * len + j];
  acc[warp][lane] = a;
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int i = 1; i < kSumWarps; ++i) a += acc[i][lane];
  gW[j] = __float2bfloat16_rn(a);
}

int64_t token_tiles(int64_t T) { return (T + kTok - 1) / kTok; }
int column_blocks(int nC) { return (nC + kCols - 1) / kCols; }
// Blocks that share a column range: together they fill the SMs.
int token_splits(int64_t T, int nC) {
  const int64_t fill = std::max(1, kBlocksPerSm * sm_count() / column_blocks(nC));
  return int(std::min(token_tiles(T), fill));
}

}  // namespace

int64_t k1_bwd_q8_any_workspace_bytes(int64_t T, int nC) {
  const int64_t n = token_splits(T, nC);
  return n == 1 ? 256 : (n * kD * nC * 4 + 255) & ~int64_t(255);
}

// codes 4-byte, go and proj 16-byte, gx 8-byte aligned.
void launch_k1_bwd_q8_any(const void *go, const void *codes, const void *scales, int fmt,
                          const void *W, const void *proj, const float *inv_rms, void *gx,
                          void *gW, float *ws, int64_t T, int nC, cudaStream_t s) {
  const int n = token_splits(T, nC);
  FMHC_DISPATCH_FMT(fmt, {
    auto k = nC % 16 ? k1_bwd_q8_any_kernel<FMT, false> : k1_bwd_q8_any_kernel<FMT, true>;
    allow_smem(reinterpret_cast<const void *>(k), sizeof(AnySmem));
    launch(k, dim3(column_blocks(nC), n), dim3(32 * kWarps), sizeof(AnySmem), s, (const bf16 *)go,
           (const uint8_t *)codes, (const uint8_t *)scales, (const bf16 *)W, (const bf16 *)proj,
           inv_rms, (bf16 *)gx, (bf16 *)gW, ws, T, nC, token_tiles(T));
  });
  if (n > 1)
    launch(k1_dw_sum_kernel, dim3(unsigned(nC)), dim3(32 * kSumWarps), 0, s, (const float *)ws,
           (bf16 *)gW, n, int64_t(kD) * nC);
}

}  // namespace fmhc
