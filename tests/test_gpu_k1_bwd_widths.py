"""K1's backward at widths for which the tensor-core kernels have no work split (C = 4768, 5152, 9536, ...)."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from flash_mhc import MHCLiteBlock, act8

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device"),
]

ops = torch.ops.flash_mhc
BF = torch.bfloat16


def _randn(*shape):
    return torch.randn(*shape, device="cuda", dtype=BF)


@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
@pytest.mark.parametrize("T,C", [(40, 4768), (64, 4768), (200, 5152), (130, 9536), (64, 4736), (33, 37920)])
def test_projection_backward(T, C, fmt):
    """Around the tensor-core kernel's smallest work (T > 32, 4 T C > 2^20), and a width with a split beside it."""
    n = 4 * C
    torch.manual_seed(T + C)
    x, W = _randn(T, 4, C), _randn(32, n) * 0.05
    go, proj, inv = _randn(T, 32), _randn(T, 32), torch.rand(T, device="cuda") + 0.5
    if fmt is None:
        x8 = x.view(T, n).double()
        gx, gW = ops.fused_rmsnorm_project_backward(go, x.view(T, n), W, proj, inv)
        assert torch.equal(ops.fused_rmsnorm_project_bwd_dx(go, x.view(T, n), W, proj, inv), gx)
    else:
        xc, xs = act8.quantize(x, fmt)
        x8 = act8.dequantize(xc, xs, torch.float32).view(T, n).double()
        gx, gW = ops.fused_rmsnorm_project_backward_q8(go, xc, xs, W, proj, inv)
    r, g, p, w = inv.double()[:, None], go.double(), proj.double(), W.double()
    want = r * (g @ w) - (g * p).sum(1, keepdim=True) * r * r / n * x8
    # One bf16 rounding (2^-8 of the value), and f32 sums of 32 products with a few more steps: at most 40
    # roundings, 2^-24 of the terms' magnitude each, doubled for products of rounded factors.
    mag = r * (g.abs() @ w.abs()) + (g * p).abs().sum(1, keepdim=True) * r * r / n * x8.abs()
    assert ((gx.view(T, n).double() - want).abs() <= want.abs() * 2**-8 + mag * 40 * 2.0**-23 + 1e-30).all()
    gos = (go.float() * inv[:, None]).to(BF).double()
    want = gos.t() @ x8
    lim = want.abs() * 2**-8 + (gos.abs().t() @ x8.abs()) * ((T + 8) * 2.0**-23) + 1e-30
    assert ((gW.double() - want).abs() <= lim).all()


@pytest.mark.parametrize("fmt", [None, "int8"])
def test_block_trains(fmt):
    T, C = 64, 4768
    torch.manual_seed(3)
    blk = MHCLiteBlock(4, C, nn.Identity(), checkpoint_format=fmt).cuda().to(BF)
    x = _randn(T, 4, C).requires_grad_()
    blk(x).float().square().sum().backward()
    for t in (x, blk.W_all.weight, blk.W_all.bias):
        assert torch.isfinite(t.grad).all() and t.grad.any()
