"""8-bit rows and layers on a GPU where they can go wrong: values between two codes, scales at the ends of f32's range,
other types, one lost copy.  u = 2^-24."""

from __future__ import annotations

import copy

import numpy as np
import pytest
import torch
import torch.nn as nn

from flash_mhc import _native, int8, norm

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device"),
]

U = 2.0 ** -24
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("C", [64, 200, 1023, 2048, 4096, 9000])
def test_codes_are_the_formats_to_the_bit(C, dtype):
    """Those between two steps among them (x = a / 2 is 63.5 steps), in the kernels and in torch on both devices."""
    x = torch.randn(2000, C, generator=_gen(C), device="cuda").to(dtype)
    x[:, 7] = x.float().abs().amax(-1).to(dtype)
    x[:, 8] = x[:, 7] / 2
    codes, scales = int8.quantize_rows(x)
    v = x.float().cpu().numpy()
    a = np.abs(v).max(-1)
    assert np.array_equal(scales.cpu().numpy(), a / np.float32(127))
    assert np.array_equal(codes.cpu().numpy(), np.rint(v * (np.float32(127) / a)[:, None]).astype(np.int8))
    for t in (x, x.cpu()):
        c, s = int8._quantize_plain(t)
        assert torch.equal(c.to(codes.device), codes) and torch.equal(s.to(scales.device), scales)


# rows of a warp, of a team of warps, of several rows per warp, of an odd width; past the widths of the other kernels
@pytest.mark.parametrize("C", [256, 2048, 4096, 64, 1023, 9000])
@pytest.mark.parametrize("size,weight", [(1e17, 3e-27), (1e-10, 1e36)])
def test_a_norm_to_8_bits_whose_weight_is_far_from_one(C, size, weight):
    """rstd w is 3e-44 or 1e39, out of f32's range, where the normalised values and their products with w are not."""
    x = (torch.randn(40, C, generator=_gen(C), device="cuda") * size).clamp(-4 * size, 4 * size)
    w = torch.linspace(1, 2, C, device="cuda") * weight
    y = x.double() / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    a = y.abs().amax(-1)
    for codes, scales, *_ in (int8.rms_norm_int8(x, w), int8.add_rms_norm_int8(x, torch.zeros_like(x), w)):
        # the sum of squares (C u, its mean's 3 u), the square root's 2 u, two products and the division: C + 8 roundings
        rel = (C + 8) * U
        assert ((scales.double() - a / 127).abs() <= rel * a / 127).all()
        assert ((codes.double() - y * (127 / a)[:, None]).abs() <= 0.5 + 2 * 127 * rel).all()
