"""The work split of K1's tensor-core backward for every width: a grid that covers it, or none said so.

Compiles the plan's header (plain C++) with the host compiler and walks over the widths."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "flash-mhc_b200" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include "k1_bwd_plan.h"
using namespace fmhc::k1tc;
// nC, T, has, G, ngroups, grid, base, rem, nkc, ntt, bytes of the plans of every width up to 4 x 40000 columns.
int main() {
  const long long tokens[] = {1, 128, 129, 4096, 65536, 1ll << 31};
  for (long long C = 32; C <= 40000; C += 32)
    for (long long T : tokens) {
      const BwdPlan p = bwd_plan(T, 4 * C, 148);
      printf("%lld %lld %d %d %d %d %d %d %d %d %lld\n", 4 * C, T, int(bwd_has_plan(T, 4 * C, 148)), p.G, p.ngroups,
             p.grid, p.base, p.rem, p.nkc, p.ntt, (long long)p.part_bytes);
    }
  // no plan at all: no tokens, other widths, no device
  printf("%d %d %d %d\n", bwd_has_plan(0, 4096, 148), bwd_has_plan(8, 4000, 148), bwd_has_plan(8, 0, 148),
         bwd_has_plan(8, 4096, 0));
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host C++ compiler")
def test_every_width_has_a_covering_plan_or_says_that_it_has_none(tmp_path):
    (tmp_path / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", "-o", str(tmp_path / "plan"),
                    str(tmp_path / "plan.cpp")], check=True)
    lines = subprocess.run([str(tmp_path / "plan")], check=True, capture_output=True, text=True).stdout.splitlines()
    assert lines.pop() == "0 0 0 0"
    without = set()
    for line in lines:
        nC, T, has, G, ngroups, grid, base, rem, nkc, ntt, part = map(int, line.split())
        possible = any(nkc % g == 0 and nkc // g <= 148 for g in (8, 4, 2, 1))
        assert has == possible, line
        if not has:
            without.add(nC // 4)
            continue
        assert G in (1, 2, 4, 8) and G * ngroups == nkc and nkc * 128 == nC and (ntt - 1) * 128 < T <= ntt * 128, line
        # every group has a CTA, and the groups' CTAs are the grid
        assert base >= 1 and 0 <= rem < ngroups and base * ngroups + rem == grid <= 148, line
        assert part >= grid * G * 32 * 128 * 4, line
    assert {4768, 4832, 5152, 9536, 37920} <= without and not {1024, 4736, 8192, 18944, 37888} & without
