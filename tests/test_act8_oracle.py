"""The 8-bit format's oracle against its own definition, and against torch's e4m3 (CPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import act8_oracle as A


def test_e4m3_rounding_matches_torch():
    q = torch.linspace(-448, 448, 40001, dtype=torch.float64)
    q = torch.cat([q, q / 448 * 0.03, torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9])])
    want = q.float().to(torch.float8_e4m3fn).double()
    assert np.array_equal(A.e4m3_round(q.float().double().numpy()), want.numpy())


@pytest.mark.parametrize("fmt,half", [("int8", 2.0 ** -1), ("e4m3", None)])
def test_quantize_restore_error_is_at_most_half_a_step(fmt, half):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((40, 77)).astype(np.float32) * np.exp(rng.standard_normal((40, 1)) * 8)
    codes, scales = A.quantize(x, fmt)
    s = np.exp2(np.repeat(scales.astype(np.float64), 32, axis=-1)[:, :77] - 127)
    err = np.abs(A.restore(codes, scales) - x.astype(np.float64))
    lim = s * half if fmt == "int8" else np.maximum(np.abs(x) * 2.0 ** -4, s * 2.0 ** -10)
    assert (err <= lim).all()
    assert (np.abs(codes) <= A.MOST[fmt]).all()
    # the smallest scale that fits: half of it would not hold the block's largest value
    a = np.abs(A._blocks(x)).max(-1)
    assert (a > A.MOST[fmt] * np.exp2(scales.astype(np.float64) - 128))[scales > 0].all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_edges_of_the_format(fmt):
    x = np.zeros((5, 64), dtype=np.float32)
    x[1, 3] = np.inf
    x[2, 40] = np.nan
    x[3, 0] = np.finfo(np.float32).max
    x[4, 0] = np.finfo(np.float32).smallest_subnormal
    codes, scales = A.quantize(x, fmt)
    assert scales[0].tolist() == [0, 0] and not codes[0].any()
    assert scales[1].tolist() == [255, 0] and scales[2].tolist() == [0, 255]
    assert not codes[1].any() and not codes[2].any()
    r = A.restore(codes, scales)
    assert np.isnan(r[1, :32]).all() and not r[1, 32:].any()
    assert scales[3, 0] == A.TOP_SCALE[fmt] and codes[3, 0] == A.MOST[fmt]
    assert np.isfinite(np.float32(r[3, 0]))
    assert scales[4, 0] == 0
