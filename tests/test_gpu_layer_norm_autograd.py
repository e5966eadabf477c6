"""The norm's autograd: broadcast gradients with every checkpoint, and what requires a gradient when parts are frozen."""

from __future__ import annotations

import itertools

import pytest
import torch

from flash_mhc import act8, norm

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device"),
]

ops = torch.ops.flash_mhc
EPS = 1e-5
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _inputs(rows, C, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows * 10007 + C)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    return r(rows, C) * 3 + 1, r(rows, C), r(C), r(C)


def _backward(g, x, mean, rstd, w, b, fmt):
    """The backward op with a dense gradient: what autograd has to give for an expanded one, to the bit."""
    if fmt is None:
        return ops.layer_norm_backward(g, x, mean, rstd, w, b)
    return ops.layer_norm_backward_q8(g, *act8.quantize(x, fmt), mean, rstd, w, b)


@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,C", [(1, 1), (37, 264), (1030, 77), (200, 4096)])
def test_broadcast_gradients(rows, C, dtype, fmt):
    """A sum's gradient is one number expanded over y, a sum over rows' one row expanded, a sum over columns' one
    column: strides of zero in either dimension."""
    x, g, w, b = _inputs(rows, C, dtype)
    _, mean, rstd = ops.layer_norm(x, w, b, EPS)
    for grad in (torch.ones((), device="cuda", dtype=dtype).expand(rows, C), g[:1].expand(rows, C), g[:, :1].expand(rows, C)):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        norm.layer_norm(*leaves, EPS, fmt).backward(grad)
        for leaf, want in zip(leaves, _backward(grad.contiguous(), x, mean, rstd, w, b, fmt)):
            assert torch.equal(leaf.grad, want)
    # what a user writes
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    norm.layer_norm(*leaves, EPS, fmt).sum().backward()
    for leaf, want in zip(leaves, _backward(torch.ones_like(x), x, mean, rstd, w, b, fmt)):
        assert torch.equal(leaf.grad, want)


@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
def test_what_requires_a_gradient(fmt):
    """y requires a gradient exactly where x, weight or bias does and gradients are enabled; each that does gets its
    own, the others none."""
    x, g, w, b = _inputs(40, 264, torch.bfloat16)
    _, mean, rstd = ops.layer_norm(x, w, b, EPS)
    want = _backward(g, x, mean, rstd, w, b, fmt)
    for wants in itertools.product((False, True), repeat=3):
        leaves = [t.clone().requires_grad_(r) for t, r in zip((x, w, b), wants)]
        with torch.no_grad():
            assert not norm.layer_norm(*leaves, EPS, fmt).requires_grad
        y = norm.layer_norm(*leaves, EPS, fmt)
        assert y.requires_grad == any(wants)
        outs = ops.layer_norm(*leaves, EPS) if fmt is None else ops.layer_norm_q8(*leaves, EPS, fmt)
        assert [t.requires_grad for t in outs] == [any(wants)] + [False] * (len(outs) - 1)
        if any(wants):
            y.backward(g)
        for leaf, r, grad in zip(leaves, wants, want):
            assert (leaf.grad is not None) == r and (not r or torch.equal(leaf.grad, grad))
