"""Layer norm's backward of many rows per warp: each row with its own statistics and scale bytes."""

from __future__ import annotations

import pytest
import torch

import flash_mhc  # noqa: F401
from flash_mhc import norm  # noqa: F401

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device"),
]

ops = torch.ops.flash_mhc
BF = torch.bfloat16


@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
@pytest.mark.parametrize("rows,width", [(30001, 64), (30001, 256), (20000, 264), (9000, 1024), (5000, 2048), (3000, 4104)])
def test_rows_do_not_see_one_another(rows, width, fmt):
    """A warp holds the statistics and scale bytes of three rows at a time, each copied by a few of its lanes.

    Neighbouring rows differ in size by up to 2^40 and in mean, so a row that used another's would show; a row's
    gradient has the same bits wherever the row stands, so the rows in reverse give the gradients in reverse."""
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    size = torch.exp2(torch.randint(-20, 21, (rows, 1), generator=g, device="cuda").float())
    x = ((torch.randn(rows, width, generator=g, device="cuda") + torch.randn(rows, 1, generator=g, device="cuda")) * size).to(BF)
    gy = torch.randn(rows, width, generator=g, device="cuda").to(BF)
    w = torch.randn(width, generator=g, device="cuda").to(BF)

    def backward(x, gy):
        if fmt is None:
            _, mean, rstd = ops.layer_norm(x, w, None, 0.0)
            return ops.layer_norm_backward(gy, x, mean, rstd, w, None)[0], x, mean, rstd
        _, mean, rstd, c, s = ops.layer_norm_q8(x, w, None, 0.0, fmt)
        x8 = ops.act_dequantize(c, s, torch.float32)
        return ops.layer_norm_backward_q8(gy, c, s, mean, rstd, w, None)[0], x8, mean, rstd

    gx, read, mean, rstd = backward(x, gy)
    assert torch.equal(backward(x.flip(0), gy.flip(0))[0], gx.flip(0))
    # and the formula's, in 64 bits: one bf16 rounding, and f32 sums of `width` values (a lane adds at most 128 of
    # them, then ten levels): below 200 roundings of 2^-24, 1.2e-5 of the terms' magnitude
    M, R, G, X = mean.double()[:, None], rstd.double()[:, None], gy.double() * w.double(), read.double()
    xh = (X - M) * R
    c2 = (G * xh).mean(-1, keepdim=True)
    want = R * (G - G.mean(-1, keepdim=True) - xh * c2)
    mag = R * (G.abs() + G.abs().mean(-1, keepdim=True) + xh.abs() * (G * xh).abs().mean(-1, keepdim=True))
    assert ((gx.double() - want).abs() <= want.abs() * 2**-8 + 1.2e-5 * mag).all()
