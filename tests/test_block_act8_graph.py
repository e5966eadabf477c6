"""MHCLiteBlock(checkpoint_format=) quantises only where a graph is recorded, eagerly and compiled."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

from flash_mhc import MHCLiteBlock, act8

BF = torch.bfloat16
T, C = 10, 64
gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


class Ops(TorchDispatchMode):
    """The names of this package's ops that are called."""

    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace == "flash_mhc":
            self.names.append(func._opname)
        return func(*args, **(kwargs or {}))


class Scaled(nn.Module):
    """A layer with a parameter that may also be handed a tensor."""

    def __init__(self):
        super().__init__()
        self.w = nn.Parameter(torch.ones(C))

    def forward(self, x, scale=None):
        return x * self.w if scale is None else x * self.w * scale


def block(fmt, device="cuda"):
    torch.set_default_dtype(BF)  # made where it stays, since a fake module cannot be moved
    try:
        with torch.device(device):
            return MHCLiteBlock(4, C, Scaled(), checkpoint_format=fmt)
    finally:
        torch.set_default_dtype(torch.float32)


def check_which_ops_run(fmt, make):
    """``make()``: a block and its x on the (maybe fake) device."""
    q8 = lambda names: [n for n in names if n.endswith("_q8") or n.startswith("act_")]  # noqa: E731

    def forward(blk, x, **kwargs):
        with Ops() as seen:
            out = blk(x, **kwargs)
        return out, seen.names

    blk, x = make()
    blk.requires_grad_(False)
    out, names = forward(blk, x)
    assert not out.requires_grad and names and not q8(names)
    # A tensor that only the layer sees: x is quantised for K4's backward, once the graph begins.
    scale = torch.ones(C, device=x.device, dtype=BF, requires_grad=True)
    out, names = forward(blk, x, scale=scale)
    assert out.requires_grad and q8(names) == ["act_quantize", "fused_post_res_q8"]
    assert q8(forward(blk, x, scale=scale.detach())[1]) == []
    # x, a mixing parameter or the layer's parameter alone: the forward that writes the codes.
    for wants in (x, blk.alpha_res, blk.layer.w):
        wants.requires_grad_(True)
        out, names = forward(blk, x)
        assert out.requires_grad and q8(names) == ["mhc_pre_forward_q8", "fused_post_res_q8"]
        wants.requires_grad_(False)
    # A tensor in a parameter's place, as sharding wrappers put there.
    w = torch.zeros_like(blk.W_all.weight).requires_grad_()
    del blk.W_all.weight
    blk.W_all.weight = w * 2
    out, names = forward(blk, x)
    assert out.requires_grad and q8(names) == ["mhc_pre_forward_q8", "fused_post_res_q8"]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_ops_that_run_fake(fmt):
    with FakeTensorMode():
        check_which_ops_run(fmt, lambda: (block(fmt), torch.zeros(T, 4, C, dtype=BF, device="cuda")))


@pytest.mark.parametrize("fmt", [pytest.param(f, marks=gpu) for f in ("int8", "e4m3")])
def test_ops_that_run(fmt):
    check_which_ops_run(fmt, lambda: (block(fmt), torch.randn(T, 4, C, dtype=BF, device="cuda")))


@pytest.mark.parametrize("fmt", [pytest.param(f, marks=gpu) for f in ("int8", "e4m3")])
def test_gradient_of_a_tensor_that_only_the_layer_sees(fmt):
    """It is that of the block whose graph begins at x: K4's backward reads the same codes."""
    x, g = torch.randn(T, 4, C, device="cuda").to(BF), torch.randn(T, 4, C, device="cuda").to(BF)
    got = []
    blk = block(fmt).requires_grad_(False)
    for x_grad in (False, True):
        scale = torch.full((C,), 0.5, device="cuda", dtype=BF, requires_grad=True)
        out = blk(x.clone().requires_grad_(x_grad), scale=scale)
        out.backward(g)
        got.append((out.detach(), scale.grad))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and got[0][1].any()


@pytest.mark.parametrize("fmt", [pytest.param(f, marks=gpu) for f in (None, "int8", "e4m3")])
def test_compiled(fmt, monkeypatch):
    """A compiled step has the eager step's bits; a compiled no-grad forward quantises nothing."""
    launched = []
    launch = act8._launch
    monkeypatch.setattr(act8, "_launch", lambda t, name, *args: (launched.append(name), launch(t, name, *args))[1])
    blk = block(fmt)
    f = torch.compile(blk, backend="aot_eager")
    x, g = torch.randn(T, 4, C, device="cuda").to(BF), torch.randn(T, 4, C, device="cuda").to(BF)
    with torch.no_grad():
        want = blk(x)
        assert torch.equal(f(x), want) and not launched
    # in the order of the model's tensors, and with the streams in another order in memory
    for order in (lambda t: t, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)):
        res = []
        for call in (blk, f):
            blk.zero_grad(set_to_none=True)
            xr = order(x.clone()).requires_grad_()
            out = call(xr)
            out.backward(g)
            res.append((out.detach(), xr.grad, [p.grad for p in blk.parameters()]))
        assert torch.equal(res[0][0], want) and torch.equal(res[1][0], want)
        assert torch.equal(res[0][1], res[1][1]) and all(map(torch.equal, res[0][2], res[1][2]))
    assert any("q8" in n for n in launched) == (fmt is not None)


def test_a_block_pickled_before_the_argument_existed():
    """A whole module that was saved without the attribute runs as one without a format."""
    with FakeTensorMode():
        blk = block("int8")
        del blk.__dict__["checkpoint_format"]
        with Ops() as seen:
            out = blk(torch.zeros(T, 4, C, dtype=BF, device="cuda", requires_grad=True))
    assert out.requires_grad and seen.names == ["mhc_pre_forward", "fused_post_res"]
