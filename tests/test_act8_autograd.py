"""Backward through the 8-bit ops: refused with a message, never a gradient that goes missing."""

from __future__ import annotations

import warnings

import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode

from flash_mhc import MHCLiteBlock, act8

ops = torch.ops.flash_mhc
BF, U8 = torch.bfloat16, torch.uint8
T, n, C, NB = 6, 4, 64, 2


def calls(fmt, device):
    """name -> arguments; every floating tensor among them requires a gradient."""
    ct = act8.FORMATS[fmt][1]
    f = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=device, requires_grad=True)  # noqa: E731
    x, lo, W = f(T, n, C, dtype=BF), f(T, C, dtype=BF), f(32, n * C, dtype=BF)
    h, H, p32, inv, a = f(T, n), f(T, n, n), f(T, 32, dtype=BF), f(T), f(1)
    xc, xs = torch.zeros(T, n, C, dtype=ct, device=device), torch.zeros(T, n, NB, dtype=U8, device=device)
    lc, ls = torch.zeros(T, C, dtype=ct, device=device), torch.zeros(T, NB, dtype=U8, device=device)
    return {
        "fused_pre_map_q8": (x, h, fmt),
        "fused_post_res_q8": (x, lo, H, h, fmt),
        "mhc_pre_forward_q8": (x, W, a, a, a, f(32), f(24, 16), fmt),
        "pre_map_grad_h_q8": (lo, xc, xs),
        "post_res_grad_params_q8": (x, xc, xs, lc, ls, h),
        "fused_rmsnorm_project_backward_q8": (p32, xc, xs, W, p32, inv),
    }


def check(fmt, device):
    for name, args in calls(fmt, device).items():
        outs = getattr(ops, name)(*args)
        outs = outs if isinstance(outs, (tuple, list)) else (outs,)
        with torch.no_grad():
            alone = getattr(ops, name)(*args)
        assert not any(t.requires_grad for t in (alone if isinstance(alone, (tuple, list)) else (alone,)))
        for t in outs:
            kept = t.dtype not in (torch.float32, BF)  # codes and scales are outside autograd
            assert t.requires_grad != kept, (name, t.dtype)
            if not kept:
                with pytest.raises(RuntimeError, match=f"{name} has no derivative"):
                    t.float().sum().backward(retain_graph=True)
        assert all(t.grad is None for t in args if isinstance(t, torch.Tensor)), name
    x = args[0].new_zeros(T, C).requires_grad_()
    codes, scales = ops.act_quantize(x, fmt)
    assert not codes.requires_grad and not scales.requires_grad
    if fmt == "e4m3":  # codes of a floating type can be told to require a gradient
        codes.requires_grad_()
    assert not ops.act_dequantize(codes, scales, BF).requires_grad


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_backward_raises_with_fake_tensors(fmt):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with FakeTensorMode():
            check(fmt, "cpu")


gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


@pytest.mark.parametrize("fmt", [pytest.param(f, marks=gpu) for f in ("int8", "e4m3")])
def test_backward_raises(fmt):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        check(fmt, "cuda")


@pytest.mark.parametrize("fmt", [pytest.param(f, marks=gpu) for f in ("int8", "e4m3")])
def test_forward_mode_is_refused(fmt):
    x, h = torch.randn(T, n, C, device="cuda", dtype=BF), torch.rand(T, n, device="cuda")
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(h, torch.ones_like(h))
        with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            ops.fused_pre_map_q8(x, dual, fmt)
        assert torch.equal(ops.fused_pre_map_q8(x, h, fmt)[0], ops.fused_pre_map(x, h))


@pytest.mark.parametrize("fmt", [pytest.param(f, marks=gpu) for f in ("int8", "e4m3")])
def test_the_block_still_differentiates(fmt):
    torch.manual_seed(0)
    blk = MHCLiteBlock(4, C, nn.Linear(C, C), checkpoint_format=fmt).cuda().to(BF)
    x = torch.randn(T, 4, C, device="cuda", dtype=BF).requires_grad_()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        blk(x).float().square().sum().backward()
    assert x.grad.any() and all(p.grad is not None for p in blk.parameters())
