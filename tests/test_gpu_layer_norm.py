"""GPU parity of layer norm, with its input kept as it is and in 8 bits, against the float64 oracle.

Tolerances.  u = 2^-24.  The kernels add a row in chains of at most
D = 45 + C / 256 additions (per lane, across the warp, across the warps), so a
row's sum is off by at most D u times the sum of the magnitudes, whatever the
order.  A column's sum over the rows is off by at most (rows + 16) u times the
sum of its magnitudes.  An output in a 16-bit type adds half a step, eps / 2 of
its value (and half the smallest f16 subnormal).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch
import torch.nn as nn

from flash_mhc import act8, norm
from oracle import act8_oracle as A

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device"),
]

ops = torch.ops.flash_mhc
U = 2.0 ** -24
EPS = 1e-5
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
# one value, ragged, odd; the widths at which a warp, two chunks and a team fill
# up or spill over; widths past the register kernels
WIDTHS = [1, 2, 8, 31, 40, 256, 264, 1000, 1023, 1024, 1032, 2048, 4104, 8192, 8200, 20000]


def _np(t):
    return t.detach().float().double().cpu().numpy()


def _half(dtype, v):
    if dtype == F32:
        return 2 * U * np.abs(v)
    return torch.finfo(dtype).eps / 2 * np.abs(v) + (2.0 ** -25 if dtype == HF else 0.0)


def _inputs(rows, C, dtype, pdt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 101 + rows * 17 + C)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = (r(rows, C) * torch.exp(r(rows, 1)) + 0.7 * r(C)).to(dtype)
    return x, r(rows, C).to(dtype), (1 + 0.3 * r(C)).to(pdt), (0.2 * r(C)).to(pdt)


def _within(name, got, want, bound):
    assert tuple(got.shape) == tuple(want.shape), name
    v = _np(got)
    if got.dtype == HF:
        # 65504 is the largest f16 and 65520 the first number that rounds to
        # infinity: beyond it infinity is the right result.
        full = (np.abs(want) >= 65520.0) & (v == np.copysign(np.inf, want))
        v, want = np.where(full, 0.0, v), np.where(full, 0.0, want)
    over = np.abs(v - want) - bound
    worst = over.max() if over.size else 0.0
    assert worst <= 0, f"{name}: {worst:.3g} over the bound"


def _check_forward(x, w, b, eps, y, mean, rstd):
    C = x.shape[-1]
    D = 45 + C / 256
    v = _np(x)
    want, m, r = A.layer_norm_fwd(v, None if w is None else _np(w), None if b is None else _np(b), eps)
    mb = D * U * np.abs(v).mean(-1) + U * np.abs(m)
    _within("mean", mean, m, mb)
    # the variance about a mean that is off by mb is off by mb^2 and its own D u
    var = np.square(v - m[..., None]).mean(-1)
    rel = 0.5 * ((D + 8) * U * var + mb * mb) / (var + eps) + 4 * U
    _within("rstd", rstd, r, rel * r + 1e-30)
    aw = 1.0 if w is None else np.abs(_np(w))
    xh = np.abs((v - m[..., None]) * r[..., None])
    off = aw * (xh * (rel + 4 * U)[..., None] + (mb * r)[..., None])
    _within("y", y, want, off + 2 * U * np.abs(want) + (0 if b is None else 2 * U * np.abs(_np(b)))
            + _half(x.dtype, np.abs(want) + off))


def _check_backward(g, x_read, mean, rstd, w, grads, params):
    C, rows = x_read.shape[-1], x_read.size // x_read.shape[-1]
    (gx, gw, gb), (sx, sw, sb) = A.layer_norm_bwd(_np(g), x_read, _np(mean), _np(rstd), None if w is None else _np(w))
    off = (45 + C / 256 + 16) * U * sx
    _within("grad_x", grads[0], gx, off + _half(g.dtype, np.abs(gx) + off) + 1e-30)
    for name, got, want, s in (("grad_weight", grads[1], gw, sw), ("grad_bias", grads[2], gb, sb)):
        if got is None or not got.numel():
            continue
        off = (rows + 16) * U * s
        _within(name, got, want, off + _half(params, np.abs(want) + off) + 1e-30)


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("dtype,pdt", [(BF, BF), (BF, F32), (HF, HF), (F32, F32), (F32, BF)])
def test_forward_and_backward(C, dtype, pdt):
    for rows in (1, 5, 67) if C > 1100 else (1, 5, 67, 700):
        x, g, w, b = _inputs(rows, C, dtype, pdt)
        y, mean, rstd = ops.layer_norm(x, w, b, EPS)
        assert y.dtype == dtype and mean.dtype == rstd.dtype == F32
        _check_forward(x, w, b, EPS, y, mean, rstd)
        grads = ops.layer_norm_backward(g, x, mean, rstd, w, b)
        assert [t.dtype for t in grads] == [dtype, pdt, pdt]
        _check_backward(g, _np(x), mean, rstd, w, grads, pdt)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("dtype,pdt", [(BF, BF), (HF, F32), (F32, F32)])
def test_from_an_8_bit_input(C, dtype, pdt, fmt):
    for rows in (1, 67):
        x, g, w, b = _inputs(rows, C, dtype, pdt)
        y, mean, rstd, codes, scales = ops.layer_norm_q8(x, w, b, EPS, fmt)
        for got, want in zip((y, mean, rstd), ops.layer_norm(x, w, b, EPS)):
            assert torch.equal(got, want)
        want_c, want_s = A.quantize(_np(x), fmt)
        assert np.array_equal(scales.cpu().numpy(), want_s)
        assert np.array_equal(codes.float().cpu().numpy(), want_c)
        grads = ops.layer_norm_backward_q8(g, codes, scales, mean, rstd, w, b)
        _check_backward(g, A.restore(want_c, want_s), mean, rstd, w, grads, pdt)


@pytest.mark.parametrize("which", ["none", "weight", "bias"])
@pytest.mark.parametrize("C", [40, 77])
def test_missing_parameters(C, which):
    x, g, w, b = _inputs(33, C, BF, F32)
    w, b = (w if which == "weight" else None), (b if which == "bias" else None)
    y, mean, rstd = ops.layer_norm(x, w, b, EPS)
    _check_forward(x, w, b, EPS, y, mean, rstd)
    grads = ops.layer_norm_backward(g, x, mean, rstd, w, b)
    assert [t.numel() for t in grads[1:]] == [0 if p is None else C for p in (w, b)]
    _check_backward(g, _np(x), mean, rstd, w, grads, F32)


@pytest.mark.parametrize("C", [64, 256, 512, 1024, 2048])
def test_every_number_of_rows_per_block(C):
    """Block and shared-memory sizes follow the rows per SM: one row to two waves of every team count."""
    w, b = torch.randn(C, device="cuda"), torch.randn(C, device="cuda")
    for rows in [*range(1, 30, 7), *range(100, 148 * 26, 148 * 2 - 5)]:
        x, g, _, _ = _inputs(rows, C, BF, BF)
        for ww, bb in ((w, b), (None, None)):
            y, mean, rstd = ops.layer_norm(x, ww, bb, EPS)
            gx, gw, gb = ops.layer_norm_backward(g, x, mean, rstd, ww, bb)
            xf = x.double()
            m = xf.mean(-1, keepdim=True)
            r = 1 / torch.sqrt((xf - m).square().mean(-1, keepdim=True) + EPS)
            xh = (xf - m) * r
            want = xh if ww is None else xh * ww.double() + bb.double()
            # half a bf16 step, and 1e-5 of the terms for the f32 arithmetic
            assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5 * (1 + want.abs() + xh.abs())).all()
            t = g.double() if ww is None else g.double() * ww.double()
            want = r * (t - t.mean(-1, keepdim=True) - xh * (t * xh).mean(-1, keepdim=True))
            lim = 2.0 ** -8 * want.abs() + 1e-5 * r * (1 + t.abs() + xh.abs())
            assert ((gx.double() - want).abs() <= lim).all()
            if ww is not None:
                s = (g.double() * xh).abs().sum(0)
                assert ((gw.double() - (g.double() * xh).sum(0)).abs() <= 1e-5 * s).all()
                assert ((gb.double() - g.double().sum(0)).abs() <= 1e-5 * g.double().abs().sum(0)).all()


@pytest.mark.parametrize("C", [96, 1023, 2600])
def test_statistics_of_rows_far_from_zero(C):
    """Mean 1000 times the spread: <x^2> - mean^2 would lose every digit of the variance."""
    x, g, w, b = _inputs(19, C, F32, F32)
    x = 1000.0 + torch.randn_like(x)
    y, mean, rstd = ops.layer_norm(x, w, b, EPS)
    _check_forward(x, w, b, EPS, y, mean, rstd)
    var = _np(x).var(-1)
    assert np.abs(_np(rstd) * np.sqrt(var + EPS) - 1).max() < 1e-4


def test_constant_rows_zero_rows_and_non_finite_rows():
    C = 264
    x, g, w, b = _inputs(6, C, F32, F32)
    x[0], x[1], x[3, 5], x[4, 9] = 3.0, 0.0, float("nan"), float("inf")
    y, mean, rstd = ops.layer_norm(x, w, b, EPS)
    _check_forward(x[[0, 1, 2, 5]], w, b, EPS, y[[0, 1, 2, 5]], mean[[0, 1, 2, 5]], rstd[[0, 1, 2, 5]])
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).all()
    for codes in (False, True):
        if codes:
            _, mean, rstd, c, s = ops.layer_norm_q8(x, w, b, EPS, "int8")
            gx = ops.layer_norm_backward_q8(g, c, s, mean, rstd, w, b)[0]
        else:
            gx = ops.layer_norm_backward(g, x, mean, rstd, w, b)[0]
        assert torch.isnan(gx[3]).any() and torch.isfinite(gx[[0, 1, 2, 5]]).all()


def test_no_rows():
    x, g, w, b = _inputs(0, 64, BF, F32)
    y, mean, rstd, codes, scales = ops.layer_norm_q8(x, w, b, EPS, "e4m3")
    assert y.shape == (0, 64) and scales.shape == (0, 2)
    for grads in (ops.layer_norm_backward(g, x, mean, rstd, w, b),
                  ops.layer_norm_backward_q8(g, codes, scales, mean, rstd, w, b)):
        assert grads[0].shape == (0, 64) and not grads[1].any() and not grads[2].any()


def test_layouts():
    x, g, w, b = _inputs(60, 400, BF, BF)
    flat = x.reshape(-1)
    for v in (x[:, ::2], x.t(), x[::3], flat[1:1 + 50 * 400].view(50, 400), x.view(3, 4, 5, 400), x[7],
              x[:1].expand(9, 400)):
        C = v.shape[-1]
        ww, bb = w.repeat(2)[1:1 + C], b.repeat(2)[3:3 + C]
        y, mean, rstd = ops.layer_norm(v, ww, bb, EPS)
        assert y.shape == v.shape and mean.shape == v.shape[:-1]
        _check_forward(v, ww, bb, EPS, y, mean, rstd)
        gv = torch.randn_like(v, memory_format=torch.contiguous_format)
        grads = ops.layer_norm_backward(gv, v, mean, rstd, ww, bb)
        _check_backward(gv, _np(v), mean, rstd, ww, grads, BF)


def test_autograd_and_module():
    """y, gradients and what is kept, through LayerNorm, against the ops; broadcast gradients."""
    torch.manual_seed(0)
    x0, g, w, b = _inputs(50, 264, BF, F32)
    for fmt in (None, "int8", "e4m3"):
        m = norm.LayerNorm(264, checkpoint_format=fmt, device="cuda")
        with torch.no_grad():
            m.weight.copy_(w)
            m.bias.copy_(b)
        x = x0.clone().requires_grad_(True)
        kept = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
            y = m(x)
        assert (any(t.dtype in (torch.int8, torch.float8_e4m3fn) for t in kept)) == (fmt is not None)
        assert any(t.shape == x.shape and t.dtype == BF for t in kept) == (fmt is None)
        want_y, mean, rstd = ops.layer_norm(x0, w, b, m.eps)
        assert torch.equal(y, want_y)
        y.backward(g)
        if fmt is None:
            want = ops.layer_norm_backward(g, x0, mean, rstd, w, b)
        else:
            want = ops.layer_norm_backward_q8(g, *act8.quantize(x0, fmt), mean, rstd, w, b)
        assert torch.equal(x.grad, want[0]) and torch.equal(m.weight.grad, want[1]) and torch.equal(m.bias.grad, want[2])
        # a sum's gradient is one number broadcast over y
        x.grad = None
        m(x).sum().backward()
        one = torch.ones_like(x0)
        if fmt is None:
            assert torch.equal(x.grad, ops.layer_norm_backward(one, x0, mean, rstd, w, b)[0])
        with torch.no_grad():
            assert torch.equal(m(x0), want_y)
    # a frozen input or frozen parameters get no gradient
    m = norm.LayerNorm(264, device="cuda", dtype=BF)
    m.requires_grad_(False)
    x = x0.clone().requires_grad_(True)
    m(x).backward(g)
    assert x.grad is not None and m.weight.grad is None
    assert not norm.layer_norm(x, m.weight, m.bias).detach().requires_grad
    y, mean, rstd = ops.layer_norm(x, m.weight, m.bias, EPS)
    assert y.requires_grad and not mean.requires_grad and not rstd.requires_grad


@pytest.mark.parametrize("C", [64, 257])
def test_gradients_against_differences(C):
    rows = 9
    x, g, w, b = _inputs(rows, C, F32, F32)
    y, mean, rstd = ops.layer_norm(x, w, b, EPS)
    gx, gw, gb = (_np(t) for t in ops.layer_norm_backward(g, x, mean, rstd, w, b))
    rng = np.random.default_rng(1)
    dx, dw, db = (rng.standard_normal(s) for s in ((rows, C), C, C))
    f = lambda t: (_np(g) * A.layer_norm_fwd(_np(x) + t * dx, _np(w) + t * dw, _np(b) + t * db, EPS)[0]).sum()  # noqa: E731
    diff = (f(1e-5) - f(-1e-5)) / 2e-5
    got = (gx * dx).sum() + (gw * dw).sum() + (gb * db).sum()
    # f32 gradients (2^-24 x the chains above, at most 80) and the differences' own 1e-10 x third derivatives
    lim = 80 * U * (np.abs(gx * dx).sum() + np.abs(gw * dw).sum() + np.abs(gb * db).sum()) + 1e-4 * max(1.0, abs(diff)) * 1e-2
    assert abs(got - diff) <= lim


def test_matches_torch():
    x, g, w, b = _inputs(300, 1000, F32, F32)
    ref = nn.functional.layer_norm
    xs, ws, bs = (t.clone().requires_grad_(True) for t in (x, w, b))
    ref(xs, (1000,), ws, bs, EPS).backward(g)
    xo, wo, bo = (t.clone().requires_grad_(True) for t in (x, w, b))
    norm.layer_norm(xo, wo, bo, EPS).backward(g)
    for a, r in ((xo, xs), (wo, ws), (bo, bs)):
        torch.testing.assert_close(a.grad, r.grad, atol=2e-4, rtol=2e-5)


def test_refusals():
    x, g, w, b = _inputs(4, 64, BF, BF)
    y, mean, rstd = ops.layer_norm(x, w, b, EPS)
    c, s = act8.quantize(x)
    refused = [
        lambda: ops.layer_norm(x.double(), w, b, EPS),
        lambda: ops.layer_norm(x[:, :0], None, None, EPS),
        lambda: ops.layer_norm(x, w[:32], b, EPS),
        lambda: ops.layer_norm(x, w, b.float(), EPS),
        lambda: ops.layer_norm(x, w.cpu(), b.cpu(), EPS),
        lambda: ops.layer_norm(x, w.double(), b.double(), EPS),
        lambda: ops.layer_norm(x, w, b, -1.0),
        lambda: ops.layer_norm_q8(x, w, b, EPS, "fp8"),
        lambda: norm.layer_norm(x, w, b, EPS, "fp8"),
        lambda: ops.layer_norm_backward(g, x[:2], mean, rstd, w, b),
        lambda: ops.layer_norm_backward(g, x.float(), mean, rstd, w, b),
        lambda: ops.layer_norm_backward(g, x, mean[:2], rstd, w, b),
        lambda: ops.layer_norm_backward(g, x, mean.double(), rstd, w, b),
        lambda: ops.layer_norm_backward(g, x, mean.cpu(), rstd, w, b),
        lambda: ops.layer_norm_backward_q8(g, c[:, :32], s[:, :1], mean, rstd, w, b),
        lambda: ops.layer_norm_backward_q8(g, c, s[:, :1], mean, rstd, w, b),
        lambda: ops.layer_norm_backward_q8(g, c, s.cpu(), mean, rstd, w, b),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
