// Work split of K1's tensor-core backward (k1_tc_bwd.cuh, k1_tc_bwd_q8.cuh) on a
// device of a given number of SMs, and which widths have one.  Host code only.
#pragma once

#include <stdint.h>

namespace fmhc {
namespace k1tc {

#ifndef FMHC_K1B_MAX_G  // largest group of k-chunks (TMEM holds at most 8 x 32 grad_W columns)
#define FMHC_K1B_MAX_G 8
#endif
constexpr int kBwdMaxG = FMHC_K1B_MAX_G;
static_assert(kBwdMaxG == 1 || kBwdMaxG == 2 || kBwdMaxG == 4 || kBwdMaxG == 8, "group size");
constexpr int kBwdBT = 128;  // tokens per unit (MMA M of grad_x)
constexpr int kBwdBK = 128;  // k per unit (MMA N of grad_x, M of grad_W)
constexpr int kBwdD = 32;    // projection width

struct BwdPlan {
  int ntt, nkc, G, ngroups, grid, base, rem;
  int64_t part_bytes;
};

// The nkc k-chunks form nkc / G groups, the grid's CTAs are spread over the
// groups as evenly as possible (the first `rem` groups get base + 1 CTAs, the
// rest base), and CTA i of a group of ng takes the token tiles i, i + ng, ...
// G (a divisor of nkc, at most 8) minimises an estimate of the kernel time
// fitted to measurements at nC = 4096 (T = 8192 and 65536, G = 2, 4, 8):
//   1.56 us per unit of the busiest CTA (64 KiB of HBM traffic)
// + 0.28 us per token tile of the busiest CTA (slot load and tile prep)
// + the grad_W partials, G x 16 KiB per CTA written and read back, at 6 TB/s.
// Large T favours G = 8 (fewest tile switches); small T, where the partials
// weigh more, favours smaller G.
//
// Every group needs a CTA of its own, so a width whose nkc has no divisor among
// 8, 4, 2, 1 that leaves at most `sms` groups has no plan: G and grid are 0 (on
// 148 SMs nkc = 149, the first, and every odd nkc after it; twice an odd number
// above 148; ...).  Whoever launches the kernels asks bwd_has_plan first.
inline BwdPlan bwd_plan(int64_t T, int64_t nC, int sms) {
  BwdPlan p{};
  p.ntt = int((T + kBwdBT - 1) / kBwdBT);
  p.nkc = int(nC / kBwdBK);
  double best_cost = -1.0;
  for (int G = kBwdMaxG; G >= 1; G >>= 1) {
    if (p.nkc % G) continue;
    const int ngroups = p.nkc / G;
    int64_t grid = int64_t(ngroups) * p.ntt;
    if (grid > sms) grid = sms;
    if (grid < ngroups) continue;  // every group needs a CTA
    const int base = int(grid / ngroups);
    const int64_t tiles = (p.ntt + base - 1) / base;
    const double part_us = double(grid) * G * kBwdD * kBwdBK * 4 * 2 / 6.0e6;
    const double cost = 1.56 * double(G * tiles) + 0.28 * double(tiles) + part_us;
    if (best_cost < 0 || cost < best_cost) {
      best_cost = cost;
      p.G = G;
      p.ngroups = ngroups;
      p.grid = int(grid);
      p.base = base;
      p.rem = int(grid % ngroups);
    }
  }
  p.part_bytes = (int64_t(p.grid) * p.G * kBwdD * kBwdBK * 4 + 255) & ~int64_t(255);
  return p;
}

inline bool bwd_has_plan(int64_t T, int64_t nC, int sms) {
  return T >= 1 && T <= (int64_t(1) << 31) && nC >= kBwdBK && nC % kBwdBK == 0 &&
         bwd_plan(T, nC, sms).G != 0;
}

}  // namespace k1tc
}  // namespace fmhc
