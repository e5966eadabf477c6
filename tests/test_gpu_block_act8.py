"""MHCLiteBlock with 8-bit checkpoints: outputs, gradients, what it keeps, graphs, streams, a stack of layers."""

from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from flash_mhc import MHCLiteBlock, act8
from flash_mhc.norm import LayerNorm

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device"),
]

ops = torch.ops.flash_mhc
BF = torch.bfloat16


class Layer(nn.Module):
    """What a transformer wraps: norm, two products."""

    def __init__(self, C, fmt=None):
        super().__init__()
        self.norm = LayerNorm(C, checkpoint_format=fmt)
        self.up = nn.Linear(C, 2 * C, bias=False)
        self.down = nn.Linear(2 * C, C, bias=False)

    def forward(self, x):
        return self.down(torch.nn.functional.silu(self.up(self.norm(x))))


def _block(C, fmt, seed=0, norm_fmt=None):
    torch.manual_seed(seed)
    blk = MHCLiteBlock(4, C, Layer(C, norm_fmt), checkpoint_format=fmt)
    with torch.no_grad():
        for a in (blk.alpha_pre, blk.alpha_post, blk.alpha_res):
            a.fill_(0.5)
        blk.W_all.bias.normal_(0, 0.3)
    return blk.cuda().to(BF).train()


def _run(blk, x, g):
    blk.zero_grad(set_to_none=True)
    x = x.clone().requires_grad_(True)
    out = blk(x)
    out.backward(g)
    return out.detach(), x.grad, {k: p.grad for k, p in blk.named_parameters()}


def _data(T, C, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed + T + C)
    return tuple(torch.randn(T, 4, C, generator=g, device="cuda").to(BF) for _ in range(2))


def _expected(blk, x, g, fmt):
    """The gradients composed from the bf16 ops, with x and the layer output restored from 8 bits."""
    T, _, C = x.shape
    W = blk.W_all.weight
    args = (blk.alpha_pre, blk.alpha_post, blk.alpha_res, blk.W_all.bias, blk.perm_mat)
    with torch.no_grad():
        li, proj, inv, h_pre, h_post, H = ops.mhc_pre_forward(x, W, *args)
    li.requires_grad_(True)
    lo = blk.layer(li)
    x8 = act8.dequantize(*act8.quantize(x, fmt))
    lo8 = act8.dequantize(*act8.quantize(lo.detach(), fmt))
    glo, gH, ghp = ops.post_res_grad_params(g, x8, lo8, H, h_post)
    blk.zero_grad(set_to_none=True)
    lo.backward(glo)
    gli = li.grad
    with torch.no_grad():
        gh = ops.pre_map_grad_h(gli, x8, h_pre)
        gp, ga, gb, gc, gbias = ops.mhc_coeffs_backward_split(gh, ghp, gH, proj, *args)
        gx1, gW = ops.fused_rmsnorm_project_backward(gp, x8.view(T, 4 * C), W, proj, inv)
        gx = ops.mhc_grad_x_combine_post(gx1.view(T, 4, C), gli, h_pre, g, H)
    params = {k: p.grad for k, p in blk.named_parameters()}
    params.update({"W_all.weight": gW, "W_all.bias": gbias, "alpha_pre": ga, "alpha_post": gb, "alpha_res": gc})
    return gx, params


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("T,C", [(1, 64), (37, 72), (300, 128), (1000, 256), (70, 33)])
def test_block_output_and_gradients(T, C, fmt):
    x, g = _data(T, C)
    blk = _block(C, fmt)
    want_out = _run(_block(C, None), x, g)[0]
    out, gx, grads = _run(blk, x, g)
    assert torch.equal(out, want_out)
    want_gx, want = _expected(blk, x, g, fmt)
    # The same formulas on the same values through other kernels: what differs
    # is the order of the f32 sums, so a bf16 result moves by a step (2^-7) at
    # most, and what is computed from it (K2's backward, the products) with it.
    def close(name, a, b, steps):
        scale = b.float().abs().max().item()
        err = (a.float() - b.float()).abs().max().item()
        assert err <= steps * 2.0 ** -7 * scale + 1e-12, (name, err, scale)
    close("grad_x", gx, want_gx, 2)
    assert set(grads) == set(want)
    for k in want:
        close(k, grads[k], want[k], 4)


@pytest.mark.parametrize("fmt,limit", [("int8", 0.02), ("e4m3", 0.06)])
def test_gradients_are_near_those_of_the_unrounded_block(fmt, limit):
    """Rounding to 8 bits moves an activation by up to 2^-8 of its block's largest value (int8, rms below
    2^-8 / sqrt(3) x 4) or 2^-4 of itself (e4m3, rms 2^-4 / sqrt(3) = 0.036): gradients by no more in norm."""
    x, g = _data(2000, 256)
    _, gx, grads = _run(_block(256, fmt), x, g)
    _, gx0, grads0 = _run(_block(256, None), x, g)
    for k, a, b in [("x", gx, gx0), *((k, grads[k], grads0[k]) for k in ("W_all.weight", "W_all.bias"))]:
        assert (a.float() - b.float()).norm() <= limit * b.float().norm(), k


def test_what_a_step_keeps():
    """Bytes from forward to backward: x and the layer output in 8 bits (33/32 byte a value), not 2 bytes."""
    T, C = 4096, 256

    class Scale(nn.Module):  # keeps nothing of its input's or output's size
        def __init__(self):
            super().__init__()
            self.f = 0.5

        def forward(self, x):
            return x * self.f

    def kept(fmt):
        blk = MHCLiteBlock(4, C, Scale(), checkpoint_format=fmt).cuda().to(BF)
        x = torch.randn(T, 4, C, device="cuda").to(BF).requires_grad_(True)
        stream = (x * 1.0)  # an activation of the layer before, freed if nobody keeps it
        torch.cuda.synchronize()
        out = blk(stream)
        del stream
        torch.cuda.synchronize()
        held = torch.cuda.memory_allocated()
        out.sum().backward()
        del out
        return held
    torch.cuda.empty_cache()
    diff = kept(None) - kept("int8")
    want = T * 5 * C * (2 - 33 / 32)  # x and lo
    assert diff >= 0.95 * want


def test_stack_of_blocks_graph_replay_matches_eager():
    """Norms and blocks with checkpoints, forward and backward, captured and replayed with new inputs."""
    T, C = 700, 128
    stack = nn.Sequential(_block(C, "int8", 0, "int8"), _block(C, "e4m3", 1, "int8"))
    inputs = [_data(T, C, seed) for seed in (1, 2)]

    def step(x, g):
        out = stack(x)
        (out * g).sum().backward()
        return out

    want = []
    for x0, g0 in inputs:
        stack.zero_grad(set_to_none=True)
        x = x0.clone().requires_grad_(True)
        out = step(x, g0).detach()
        want.append((out, x.grad.clone(), [p.grad.clone() for p in stack.parameters()]))
        del out, x
    sx, sg = inputs[0][0].clone().requires_grad_(True), inputs[0][1].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            stack.zero_grad(set_to_none=True)
            sx.grad = None
            step(sx, sg)
    torch.cuda.current_stream().wait_stream(s)
    stack.zero_grad(set_to_none=True)
    sx.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sx, sg).detach()
    for (x0, g0), (w_out, w_gx, w_p) in zip(inputs, want):
        with torch.no_grad():
            sx.copy_(x0)
            sg.copy_(g0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w_out) and torch.equal(sx.grad, w_gx)
        for p, w in zip(stack.parameters(), w_p):
            assert torch.equal(p.grad, w)


def test_two_streams_at_once():
    T, C = 900, 192
    blks = [_block(C, "int8", i) for i in range(2)]
    data = [_data(T, C, i) for i in range(2)]
    want = [_run(b, *d) for b, d in zip(blks, data)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for i, s in enumerate(streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got[i] = _run(blks[i], *data[i])
    torch.cuda.synchronize()
    for (o, gx, gp), (wo, wx, wp) in zip(got, want):
        assert torch.equal(o, wo) and torch.equal(gx, wx)
        assert all(torch.equal(gp[k], wp[k]) for k in wp)


def test_no_grad_and_empty_batch():
    x, g = _data(50, 64)
    blk = _block(64, "int8")
    with torch.no_grad():
        assert torch.equal(blk(x), _block(64, None)(x))
    out, gx, grads = _run(blk, x[:0], g[:0])
    assert out.shape == (0, 4, 64) and gx.shape == (0, 4, 64)
    assert not grads["W_all.weight"].any()
