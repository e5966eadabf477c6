// K1 backward from an 8-bit checkpoint of x for the widths that the tcgen05
// kernel (k1_tc_bwd_q8.cuh) does not take, C % 32 != 0: blocks of 32 then do not
// line up with its tiles, and rows of 4 C codes need not be what the TMA wants.
//
//   s       = (go . proj) inv^2 / nC
//   grad_x  = bf16( inv (go W) - s x8 )
//   grad_W  = bf16( sum over tokens of bf16(go inv)^T x8 )
//
// A block takes 256 of the nC columns and every gridDim.y-th tile of 64 tokens;
// a warp its own 32 columns of them: it widens their codes into a bf16 tile,
// feeds both products' warp-wide MMAs (m16n8k16) from it, writes grad_x over x
// and stores it, without waiting for the other warps.  Its columns of W stay in
// registers as MMA operands, its share of grad_W as accumulators.  All warps
// share go, bf16(go inv), s and inv of the tile, in two buffers, so one block
// barrier per tile is enough.  Blocks of one column range (their tokens differ)
// write partials of grad_W, which k1_dw_sum_kernel adds in order; a single one
// writes grad_W itself.
//
// Bound by the bytes (codes in, grad_x out) like the tcgen05 kernel; 32 (d) x 8 C
// flops per token are far below what these MMAs do. 
#include "act8.cuh"
#include "fmhc_launch.h"
#include "grid.cuh"

#include <algorithm>

namespace fmhc {

using namespace act8;
using bf16 = __nv_bfloat16;

namespace {

constexpr int kD = 32;                  // projection width
constexpr int kTok = 64;                // tokens per tile
constexpr int kCols = 256, kWarps = 8;  // columns per block, 32 per warp
constexpr int kXPitch = kCols + 8;      // bf16 elements; both pitches are odd
constexpr int kGPitch = kD + 8;         // multiples of 16 bytes (ldmatrix)
constexpr int kBlocksPerSm = 2;

struct AnySmem {
  bf16 x[kTok][kXPitch];       // x8, later grad_x
  bf16 go[2][kTok][kGPitch];
  bf16 gos[2][kTok][kGPitch];  // bf16(go inv)
  float2 sinv[2][kTok];
};

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
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
               "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
  const int kw = blockIdx.x * kCols + warp * 32;  // the warp's first column
  const bool active = kw < nC;                    // uniform in the warp
  // Loads and stores: eight lanes hold the 32 columns of a row, four each.
  const int row8 = lane >> 3, col = kw + (lane & 7) * 4;
  const bool in_col = col < nC;  // nC is a multiple of 4
  int block_of[WORD ? 1 : 4];    // where the codes' scale bytes lie in a row's 4 nb
#pragma unroll
  for (int i = 0; i < (WORD ? 1 : 4); ++i) {
    const int k = in_col ? col + i : 0, j = k / C;
    block_of[i] = j * nb + (k - j * C) / kBlock;
  }
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
  bf16 *const xw = &sm.x[0][warp * 32];
  int buf = 0;
  for (int64_t m = blockIdx.y; m < tiles; m += gridDim.y, buf ^= 1) {
    const int64_t t0 = m * kTok;
    // The codes of the tile, in flight while go and proj are prepared.
    uint32_t cw[kTok / 4], sc[kTok / 4];
#pragma unroll
    for (int i = 0; i < kTok / 4; ++i) {
      const int64_t t = t0 + i * 4 + row8;
      cw[i] = sc[i] = 0;
      if (in_col && t < T) {
        cw[i] = __ldcs(reinterpret_cast<const uint32_t *>(codes + t * nC + col));
        const uint8_t *s = scales + t * 4 * nb;
#pragma unroll
        for (int b = 0; b < (WORD ? 1 : 4); ++b) sc[i] |= uint32_t(__ldg(s + block_of[b])) << (8 * b);
      }
    }
    {  // four threads per token, eight of the 32 d each
      const int r = threadIdx.x >> 2, d = (threadIdx.x & 3) * 8;
      const int64_t t = t0 + r;
      uint4 g = make_uint4(0, 0, 0, 0), p = g;
      float inv = 0.f;
      if (t < T) {
        g = __ldg(reinterpret_cast<const uint4 *>(go + t * kD + d));
        p = __ldg(reinterpret_cast<const uint4 *>(proj + t * kD + d));
        inv = __ldg(inv_rms + t);
      }
      float gf[8], pf[8], dot = 0.f;
      Elem<bf16>::widen(g, gf);
      Elem<bf16>::widen(p, pf);
#pragma unroll
      for (int k = 0; k < 8; ++k) dot = fmaf(gf[k], pf[k], dot);
      dot += __shfl_xor_sync(0xffffffffu, dot, 1);
      dot += __shfl_xor_sync(0xffffffffu, dot, 2);
#pragma unroll
      for (int k = 0; k < 8; ++k) gf[k] *= inv;
      *reinterpret_cast<uint4 *>(&sm.go[buf][r][d]) = g;
      *reinterpret_cast<uint4 *>(&sm.gos[buf][r][d]) = Elem<bf16>::narrow(gf);
      if ((threadIdx.x & 3) == 0) sm.sinv[buf][r] = make_float2(dot * (inv * inv) / float(nC), inv);
    }
    __syncthreads();
    if (active) {
#pragma unroll
      for (int i = 0; i < kTok / 4; ++i) {
        float f[4];
        decode4<FMT>(cw[i], f);
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] *= scale_value(WORD ? sc[i] & 0xffu : (sc[i] >> (8 * k)) & 0xffu);
        *reinterpret_cast<uint2 *>(xw + (i * 4 + row8) * kXPitch + (lane & 7) * 4) =
            make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
      }
      __syncwarp();
      // grad_W += gos^T x8: first operand d x tokens, second tokens x columns,
      // both from rows of tokens.
#pragma unroll
      for (int ks = 0; ks < kTok / 16; ++ks) {
        uint32_t a[2][4], b[4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
          load_matrices_t(a[i], &sm.gos[buf][ks * 16 + (mi >> 1) * 8 + mr][i * 16 + (mi & 1) * 8]);
#pragma unroll
        for (int np = 0; np < 2; ++np) {
          load_matrices_t(b, xw + (ks * 16 + (mi & 1) * 8 + mr) * kXPitch + np * 16 + (mi >> 1) * 8);
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
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[nt][k] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          uint32_t a[4];
          load_matrices(a, &sm.go[buf][mt * 16 + (mi & 1) * 8 + mr][ks * 16 + (mi >> 1) * 8]);
#pragma unroll
          for (int nt = 0; nt < 4; ++nt) mma(acc[nt], a, wf[nt][ks][0], wf[nt][ks][1]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = mt * 16 + h * 8 + (lane >> 2);
          const float2 si = sm.sinv[buf][r];
#pragma unroll
          for (int nt = 0; nt < 4; ++nt) {
            uint32_t *p = reinterpret_cast<uint32_t *>(xw + r * kXPitch + nt * 8 + (lane & 3) * 2);
            const uint32_t v = *p;
            *p = pack_bf16x2(fmaf(-si.x, bf16lo(v), si.y * acc[nt][2 * h]),
                             fmaf(-si.x, bf16hi(v), si.y * acc[nt][2 * h + 1]));
          }
        }
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kTok / 4; ++i) {
        const int64_t t = t0 + i * 4 + row8;
        if (in_col && t < T)
          __stcs(reinterpret_cast<uint2 *>(gx + t * nC + col),
                 *reinterpret_cast<const uint2 *>(xw + (i * 4 + row8) * kXPitch + (lane & 7) * 4));
      }
      __syncwarp();  // the next tile's codes go to the same place
    }
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
