"""Codes read by words: every code of a row, and no byte beside it.

Compiles the header (plain C++) with the host compiler and reads rows whose neighbours' bytes are watched."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "flash-mhc_b200" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include "code_word.h"
// C, first and last byte that were read, codes that came out wrong, zeros that did not.
int main() {
  for (int C = 1; C <= 70; ++C) {
    int lo = 1000, hi = -1000, wrong = 0, rest = 0;
    const auto at = [](int i) { return int8_t(7 * i + 1); };
    const auto read = [&](int i, int n) { lo = i < lo ? i : lo; hi = i + n - 1 > hi ? i + n - 1 : hi; };
    const auto word = [&](int i) {
      read(i, 4);
      uint32_t w = 0;
      for (int k = 0; k < 4; ++k) w |= uint32_t(uint8_t(at(i + k))) << (8 * k);
      return w;
    };
    const auto code = [&](int i) { read(i, 1); return at(i); };
    for (int i = -8; i < C + 16; i += 4) {
      uint32_t q[3];
      fmhc::code_words(i, C, word, code, q);
      for (int k = 0; k < 12; ++k) {
        const uint8_t got = uint8_t(q[k / 4] >> (8 * (k % 4)));
        if (i + k >= 0 && i + k < C) wrong += got != uint8_t(at(i + k));
        else rest += got != 0;
      }
    }
    printf("%d %d %d %d %d\n", C, lo, hi, wrong, rest);
  }
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host C++ compiler")
def test_a_row_is_read_whole_and_alone(tmp_path):
    (tmp_path / "words.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", "-o", str(tmp_path / "words"),
                    str(tmp_path / "words.cpp")], check=True)
    lines = subprocess.run([str(tmp_path / "words")], check=True, capture_output=True, text=True).stdout.splitlines()
    assert len(lines) == 70
    for line in lines:
        C, lo, hi, wrong, rest = map(int, line.split())
        assert (lo, hi, wrong, rest) == (0, C - 1, 0, 0), line


def test_restoring_reads_codes_by_it():
    source = (CSRC / "rows8.cu").read_text()
    kernel = source[source.index("row_dequantize_general_kernel"):source.index("row_quantize_any_kernel")]
    assert kernel.count("code_words(") == 1 and kernel.count("reinterpret_cast<const uint32_t *>") == 1
