"""The shared-memory limit of a kernel never shrinks, however many kernels and devices have asked for one.

Compiles grid.cuh with the host compiler against stand-ins of the runtime calls that it makes."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "flash-mhc_b200" / "csrc"
CUDA = Path("/usr/local/cuda/include")

PROGRAM = r"""
#include <cstdio>
#include <map>
#include <utility>
#include "grid.cuh"

static int device = 0, calls = 0;
static std::map<std::pair<const void *, int>, int> limit;
extern "C" {
cudaError_t CUDARTAPI cudaGetDevice(int *d) { *d = device; return cudaSuccess; }
cudaError_t CUDARTAPI cudaDeviceGetAttribute(int *v, cudaDeviceAttr, int) { *v = 148; return cudaSuccess; }
cudaError_t CUDARTAPI cudaFuncSetAttribute(const void *k, cudaFuncAttribute, int bytes) {
  ++calls;
  limit[{k, device}] = bytes;
  return cudaSuccess;
}
}

int main() {
  static char kernels[300];
  for (size_t kib : {200, 100, 41, 150, 220, 40})
    for (device = 0; device < 3; ++device)
      for (char &k : kernels) fmhc::allow_smem(&k, kib * 1024);
  for (auto &l : limit)
    if (l.second != 220 * 1024) return 1;
  printf("%zu %d\n", limit.size(), calls);  // set to 200 KiB, then to 220
}
"""


@pytest.mark.skipif(shutil.which("g++") is None or not CUDA.exists(), reason="needs a host C++ compiler and CUDA's headers")
def test_limits_only_grow(tmp_path):
    (tmp_path / "limit.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", f"-I{CUDA}", "-o", str(tmp_path / "limit"), str(tmp_path / "limit.cpp")],
                   check=True)
    out = subprocess.run([str(tmp_path / "limit")], check=True, capture_output=True, text=True).stdout
    assert out.split() == ["900", "1800"]
