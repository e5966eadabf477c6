"""Fakes of the ops give the strides of the CUDA results, which are contiguous whatever the inputs' order is."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import flash_mhc  # noqa: F401
from flash_mhc import act8, norm  # noqa: F401

ops = torch.ops.flash_mhc
BF, U8 = torch.bfloat16, torch.uint8
T, n, C, NB = 6, 4, 72, 3


def permuted(*shape, dtype=torch.float32):
    """A dense tensor of this shape whose memory runs in the opposite order of its dimensions."""
    return torch.empty(*shape[::-1], dtype=dtype).permute(*range(len(shape))[::-1])


def calls(fmt):
    ct = act8.FORMATS[fmt][1]
    x, go, lo = permuted(T, n, C, dtype=BF), permuted(T, n, C, dtype=BF), permuted(T, C, dtype=BF)
    xf, W = permuted(T, n * C, dtype=BF), permuted(32, n * C, dtype=BF)
    h, H, p32, inv = permuted(T, n), permuted(T, n, n), permuted(T, 32, dtype=BF), torch.empty(T)
    xc, xs = permuted(T, n, C, dtype=ct), permuted(T, n, NB, dtype=U8)
    lc, ls = permuted(T, C, dtype=ct), permuted(T, NB, dtype=U8)
    a, bias, perm = torch.empty(1), torch.empty(32), permuted(24, 16)
    w = torch.empty(C, 2)[:, 0]
    return {
        "act_quantize": (x, fmt), "act_dequantize": (xc, xs, BF), "fused_pre_map_q8": (x, h, fmt),
        "fused_post_res_q8": (x, lo, H, h, fmt), "mhc_pre_forward_q8": (x, W, a, a, a, bias, perm, fmt),
        "pre_map_grad_h_q8": (lo, xc, xs), "post_res_grad_params_q8": (go, xc, xs, lc, ls, h),
        "fused_rmsnorm_project_backward_q8": (p32, xc, xs, W, p32, inv),
        "layer_norm": (lo, w, w, 1e-5), "layer_norm_q8": (x, w, None, 1e-5, fmt),
        "layer_norm_backward": (lo, lo, inv, inv, w, w), "layer_norm_backward_q8": (lo, lc, ls, inv, inv, w, w),
        "fused_rmsnorm_project": (xf, W), "fused_rmsnorm_project_bwd_dx": (p32, xf, W, p32, inv),
        "fused_rmsnorm_project_backward": (p32, xf, W, p32, inv), "fused_pre_map": (x, h),
        "fused_pre_map_backward": (lo, x, h), "fused_post_res": (x, lo, H, h),
        "fused_post_res_backward": (go, x, lo, H, h), "mhc_coeffs": (p32, a, a, a, bias, perm),
        "mhc_pre_forward": (x, W, a, a, a, bias, perm), "pre_map_grad_h": (lo, x, h),
        "mhc_grad_x_combine": (x, lo, h, None), "post_res_grad_params": (go, x, lo, H, h),
        "mhc_grad_x_combine_post": (x, lo, h, go, H),
        "mhc_coeffs_backward": (h, h, H, p32, a, a, a, bias, perm),
        "mhc_coeffs_backward_split": (h, h, H, p32, a, a, a, bias, perm),
    }



@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_fakes_are_contiguous(fmt):
    with FakeTensorMode():
        for name, args in calls(fmt).items():
            outs = getattr(ops, name)(*args)
            for i, t in enumerate(outs if isinstance(outs, (tuple, list)) else (outs,)):
                assert t.is_contiguous(), (name, i, tuple(t.shape), t.stride())


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_cuda_results_have_the_fakes_strides(fmt):
    torch.manual_seed(0)
    for name, args in calls(fmt).items():
        real = [torch.zeros_like(t, device="cuda") if isinstance(t, torch.Tensor) else t for t in args]
        assert all(a.stride() == b.stride() for a, b in zip(args, real) if isinstance(a, torch.Tensor) and a.dim() > 1)
        outs = getattr(ops, name)(*real)
        with FakeTensorMode(allow_non_fake_inputs=True) as mode:
            fakes = getattr(ops, name)(*(mode.from_tensor(t) if isinstance(t, torch.Tensor) else t for t in real))
        outs, fakes = ((v if isinstance(v, (tuple, list)) else (v,)) for v in (outs, fakes))
        for i, (a, b) in enumerate(zip(outs, fakes, strict=True)):
            assert (a.shape, a.dtype, a.stride()) == (b.shape, b.dtype, b.stride()), (name, i, a.stride(), b.stride())
