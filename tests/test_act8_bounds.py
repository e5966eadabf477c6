"""How far a value may be from what its 8-bit checkpoint restores: the bounds that the header and norm.py state.

With a the largest magnitude of a block and e its scale byte, a > M 2^(e - 128) unless e = 0 (the next smaller
scale would not hold a), so half a step of int8, 2^(e - 128), is below a / 127, and half of e4m3's smallest step,
2^(e - 137), below a / (448 2^9) < a / 2^17."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import act8_oracle as A

FORMATS = ["int8", "e4m3"]


def blocks(rng, n):
    """Blocks of 32 as f32 values: random ones, ones with a largest value just above each border of a scale, and
    ones whose values span the whole range of a code."""
    x = rng.standard_normal((n, 32)) * np.exp2(rng.integers(-60, 60, (n, 1)))
    x[: n // 3, 0] = np.exp2(rng.integers(-20, 20, n // 3)) * rng.choice([63.75, 127.0, 63.5001, 224.5, 448.0], n // 3)
    x[n // 3 : n // 2] *= np.exp2(rng.integers(-24, 1, (n // 2 - n // 3, 32)))
    return x.astype(np.float32)


def check(x, restored, scales, fmt):
    x, e = x.astype(np.float64), scales.astype(np.float64)
    a = np.abs(x).max(-1, keepdims=True)
    err = np.abs(restored - x)
    assert (scales > 0).all()
    if fmt == "int8":
        assert (err <= np.exp2(e - 128)).all() and (np.exp2(e - 128) < a / 127).all()
    else:
        assert (err <= np.maximum(np.abs(x) / 16, np.exp2(e - 137))).all() and (np.exp2(e - 137) < a / 2**17).all()
    return err / a


@pytest.mark.parametrize("fmt", FORMATS)
def test_bounds(fmt):
    x = blocks(np.random.default_rng(0), 3000)
    codes, scales = A.quantize(x, fmt)
    check(x, A.restore(codes, scales), scales, fmt)


def test_bounds_are_reached():
    """int8: more than 2^-7 of the block's largest; e4m3: all of a small value."""
    x = np.zeros((1, 32), dtype=np.float32)
    x[0, :2] = 63.75, 10.5
    codes, scales = A.quantize(x, "int8")
    assert check(x, A.restore(codes, scales), scales, "int8")[0, 1] == 0.5 / 63.75 > 2.0**-7
    x[0, :2] = 448.0, 2.0**-11
    codes, scales = A.quantize(x, "e4m3")
    assert check(x, A.restore(codes, scales), scales, "e4m3")[0, 1] == 2.0**-11 / 448.0 and not codes[0, 1]


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fmt", FORMATS)
def test_bounds_of_the_kernels(fmt, dtype):
    from flash_mhc import act8

    x = torch.from_numpy(blocks(np.random.default_rng(1), 3000)).to(dtype)
    codes, scales = act8.quantize(x.cuda(), fmt)
    restored = act8.dequantize(codes, scales, torch.float32).double().cpu().numpy()
    check(x.float().numpy(), restored, scales.cpu().numpy(), fmt)
