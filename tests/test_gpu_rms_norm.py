"""GPU parity of the root-mean-square norm (float output and 8-bit output) against the float64 oracle.

Tolerances.  u = 2^-24.  A row's sum is added in chains of at most D = 45 + C / 256
additions (per lane, across the warp, across the warps): off by at most D u times
the sum of the magnitudes.  A column's sum over the rows is off by at most
(rows + 16) u times the sum of its magnitudes.  An output in a 16-bit type adds
half a step, eps / 2 of its value (and half the smallest f16 subnormal).  A code is
within 1/2 of the exact quotient plus that quotient's relative error.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch
import torch.nn as nn

from flash_mhc import int8, norm
from oracle import rms_int8_oracle as R

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device"),
]

ops = torch.ops.flash_mhc
U = 2.0 ** -24
EPS = 1e-6
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
# one value, ragged, odd; the widths at which a warp, its chunks and a team of
# warps fill up or spill over; widths past the register kernels
WIDTHS = [1, 2, 8, 31, 40, 256, 264, 1000, 1023, 1024, 1032, 2048, 2056, 4096, 4104, 8192, 8200, 16392, 20000]
TYPES = [(BF, BF), (BF, F32), (HF, HF), (F32, F32), (F32, BF)]


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
    return x, r(rows, C).to(dtype), r(rows, C).to(dtype), r(rows, C).to(dtype), (1 + 0.3 * r(C)).to(pdt)


def _within(name, got, want, bound):
    assert tuple(got.shape) == tuple(want.shape), name
    over = np.abs(_np(got) - want) - bound
    worst = over.max() if over.size else 0.0
    assert worst <= 0, f"{name}: {worst:.3g} over the bound"


def _rel(C):
    """Relative error of rstd, and of a value times rstd and the weight."""
    r = 0.5 * (45 + C / 256 + 8) * U + 4 * U
    return r, r + 4 * U


def _check_forward(v, w, y, rstd):
    want, r = R.rms_norm_fwd(_np(v), None if w is None else _np(w), EPS)
    rel_r, rel_y = _rel(v.shape[-1])
    _within("rstd", rstd, r, rel_r * r)
    _within("y", y, want, rel_y * np.abs(want) + _half(v.dtype, np.abs(want) * (1 + rel_y)) + 1e-37)


def _check_codes(want, rel, codes, scales):
    s = R.row_scales(want)
    ok = ~np.isnan(s)
    got = scales.cpu().double().numpy()
    assert np.array_equal(np.isnan(got), ~ok)
    assert (np.abs(got - s)[ok] <= (rel + 2 * U) * s[ok]).all()
    q = R.row_quotients(want)
    off = np.abs(codes.cpu().double().numpy() - q) - (0.5 + (2 * rel + 4 * U) * np.abs(q))
    assert off.size == 0 or off.max() <= 0, off.max()
    assert np.abs(q).max(initial=0) <= 127.001 and codes.abs().max() <= 127 if codes.numel() else True


def _check_backward(g, gt, v, rstd, w, grads, params):
    rows = v.numel() // v.shape[-1]
    (gx, gw), (sx, sw) = R.rms_norm_bwd(_np(g), None if gt is None else _np(gt), _np(v), _np(rstd), None if w is None else _np(w))
    off = (45 + v.shape[-1] / 256 + 16) * U * sx
    _within("grad_x", grads[0], gx, off + _half(g.dtype, np.abs(gx) + off) + 1e-30)
    if w is None:
        assert grads[1].numel() == 0
    else:
        off = (rows + 16) * U * sw
        _within("grad_weight", grads[1], gw, off + _half(params, np.abs(gw) + off) + 1e-30)


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("dtype,pdt", TYPES)
def test_forward_and_backward(C, dtype, pdt):
    for rows in (1, 5, 67) if C > 1100 else (1, 5, 67, 700, 1500):
        x, r, g, gt, w = _inputs(rows, C, dtype, pdt)
        y, rstd = ops.rms_norm(x, w, EPS)
        assert y.dtype == dtype and rstd.dtype == F32
        _check_forward(x, w, y, rstd)
        grads = ops.rms_norm_backward(g, None, x, rstd, w)
        assert [t.dtype for t in grads] == [dtype, pdt]
        _check_backward(g, None, x, rstd, w, grads, pdt)
        # behind a residual's addition: the sum is torch's, the norm is that of the rounded sum
        y2, total, rstd2 = ops.add_rms_norm(x, r, w, EPS)
        assert torch.equal(total, x + r)
        _check_forward(total, w, y2, rstd2)
        _check_backward(g, gt, total, rstd2, w, ops.rms_norm_backward(g, gt, total, rstd2, w), pdt)


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("dtype,pdt", TYPES)
def test_output_in_8_bits(C, dtype, pdt):
    rel = _rel(C)[1]
    for rows in (1, 5, 67) if C > 1100 else (1, 5, 67, 700, 1500):
        x, r, _, _, w = _inputs(rows, C, dtype, pdt, seed=1)
        codes, scales = ops.rms_norm_int8(x, w, EPS)
        assert codes.dtype == torch.int8 and scales.dtype == F32
        _check_codes(R.rms_norm_fwd(_np(x), _np(w), EPS)[0], rel, codes, scales)
        codes, scales, total = ops.add_rms_norm_int8(x, r, w, EPS)
        assert torch.equal(total, x + r)
        _check_codes(R.rms_norm_fwd(_np(total), _np(w), EPS)[0], rel, codes, scales)


@pytest.mark.parametrize("C", [64, 256, 512, 1024, 2048, 4096])
def test_every_number_of_rows_per_block(C):
    """Block and shared-memory sizes follow the rows per SM: one row to two waves of every team count."""
    w = torch.randn(C, device="cuda")
    for rows in [*range(1, 30, 7), *range(100, 148 * 26, 148 * 3 - 5)]:
        x, r, g, gt, _ = _inputs(rows, C, BF, BF)
        for ww in (w, None):
            for res in (None, r):
                if res is None:
                    (y, rstd), total, up = ops.rms_norm(x, ww, EPS), x, None
                    codes, scales = ops.rms_norm_int8(x, ww, EPS)
                else:
                    (y, total, rstd), up = ops.add_rms_norm(x, res, ww, EPS), gt
                    assert torch.equal(total, x + res)
                    codes, scales, again = ops.add_rms_norm_int8(x, res, ww, EPS)
                    assert torch.equal(again, total)
                gx, gw = ops.rms_norm_backward(g, up, total, rstd, ww)
                v = total.double()
                rs = 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)
                xh = v * rs
                want = xh if ww is None else xh * ww.double()
                # half a bf16 step, and 1e-5 of the terms for the f32 arithmetic
                assert ((y.double() - want).abs() <= (2.0 ** -8 + 1e-5) * want.abs()).all()
                s = want.abs().amax(-1) / 127
                assert ((scales.double() - s).abs() <= 1e-5 * s).all()
                q = want / s[:, None]
                assert ((codes.double() - q).abs() <= 0.5 + 1e-5 * q.abs()).all()
                t = g.double() if ww is None else g.double() * ww.double()
                want = rs * (t - xh * (t * xh).mean(-1, keepdim=True)) + (0 if up is None else up.double())
                lim = 2.0 ** -8 * want.abs() + 1e-5 * (rs * (1 + t.abs() + xh.abs()) + 5)
                assert ((gx.double() - want).abs() <= lim).all()
                if ww is not None:
                    terms = (g.double() * xh).abs().sum(0)
                    assert ((gw.double() - (g.double() * xh).sum(0)).abs() <= 1e-5 * terms).all()


@pytest.mark.parametrize("C", [264, 77])
def test_zero_rows_and_non_finite_rows(C):
    x, r, g, _, w = _inputs(7, C, F32, F32)
    x[0], x[1], x[3, 5], x[4, 9], x[6] = 3.0, 0.0, float("nan"), float("inf"), 1e-30
    fine = [0, 1, 2, 5, 6]
    y, rstd = ops.rms_norm(x, w, EPS)
    _check_forward(x[fine], w, y[fine], rstd[fine])
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).any()
    gx = ops.rms_norm_backward(g, None, x, rstd, w)[0]
    assert torch.isnan(gx[3]).any() and torch.isfinite(gx[fine]).all()
    codes, scales = ops.rms_norm_int8(x, w, EPS)
    assert torch.isnan(scales[[3, 4]]).all() and not codes[[3, 4, 1]].any()
    _check_codes(R.rms_norm_fwd(_np(x[fine]), _np(w), EPS)[0], _rel(C)[1], codes[fine], scales[fine])
    assert scales[1].item() == np.float32(R.LEAST / 127)


def test_no_rows():
    x, r, g, gt, w = _inputs(0, 72, BF, F32)
    y, total, rstd = ops.add_rms_norm(x, r, w, EPS)
    assert y.shape == total.shape == (0, 72) and rstd.shape == (0,)
    gx, gw = ops.rms_norm_backward(g, gt, total, rstd, w)
    assert gx.shape == (0, 72) and not gw.any()
    codes, scales = ops.rms_norm_int8(x, w, EPS)
    assert codes.shape == (0, 72) and scales.shape == (0,)


def test_layouts():
    x, _, _, _, w = _inputs(60, 400, BF, BF)
    flat = x.reshape(-1)
    for v in (x[:, ::2], x.t(), x[::3], flat[1:1 + 50 * 400].view(50, 400), x.view(3, 4, 5, 400), x[7],
              x[:1].expand(9, 400)):
        C = v.shape[-1]
        ww = w.repeat(2)[1:1 + C]
        r = torch.randn(*v.shape[::-1], device="cuda", dtype=BF).permute(*range(v.dim())[::-1])
        y, total, rstd = ops.add_rms_norm(v, r, ww, EPS)
        assert y.shape == v.shape and rstd.shape == v.shape[:-1] and torch.equal(total, v + r)
        _check_forward(total, ww, y, rstd)
        y, rstd = ops.rms_norm(v, ww, EPS)
        _check_forward(v, ww, y, rstd)
        _check_backward(r, r, v, rstd, ww, ops.rms_norm_backward(r, r, v, rstd, ww), BF)
        codes, scales = ops.rms_norm_int8(v, ww, EPS)
        _check_codes(R.rms_norm_fwd(_np(v), _np(ww), EPS)[0], _rel(C)[1], codes, scales)


@pytest.mark.parametrize("C", [264, 77])
def test_autograd_and_module(C):
    torch.manual_seed(0)
    x0, r0, g, gt, w = _inputs(50, C, BF, F32)
    m = norm.RMSNorm(C, device="cuda")
    with torch.no_grad():
        m.weight.copy_(w)
    x = x0.clone().requires_grad_()
    y = m(x)
    y0, rstd = ops.rms_norm(x0, w, EPS)
    assert torch.equal(y, y0)
    y.backward(g)
    want = ops.rms_norm_backward(g, None, x0, rstd, w)
    assert torch.equal(x.grad, want[0]) and torch.equal(m.weight.grad, want[1])
    # both outputs used, only y, only total; frozen parts get nothing
    y0, t0, rstd = ops.add_rms_norm(x0, r0, w, EPS)
    for use_y, use_t in ((True, True), (True, False), (False, True)):
        x, r = x0.clone().requires_grad_(), r0.clone().requires_grad_()
        m.weight.grad = None
        y, total = m(x, r)
        assert torch.equal(y, y0) and torch.equal(total, t0)
        torch.autograd.backward([t for t, u in ((y, use_y), (total, use_t)) if u], [t for t, u in ((g, use_y), (gt, use_t)) if u])
        if use_y:
            want = ops.rms_norm_backward(g, gt if use_t else None, t0, rstd, w)
            assert torch.equal(m.weight.grad, want[1])
        else:
            want = (gt, None)
            assert m.weight.grad is None
        assert torch.equal(x.grad, want[0]) and torch.equal(r.grad, want[0])
    x = x0.clone().requires_grad_()
    m.weight.grad = None
    y, total = m.requires_grad_(False)(x, r0)
    (y.float().sum() + total.float().sum()).backward()  # broadcast gradients
    one = torch.ones_like(x0)
    assert torch.equal(x.grad, ops.rms_norm_backward(one, one, t0, rstd, w)[0]) and m.weight.grad is None
    # the same tensor twice: x + x
    x = x0.clone().requires_grad_()
    y, total = norm.add_rms_norm(x, x, w)
    y.backward(g)
    _, tt, rr = ops.add_rms_norm(x0, x0, w, EPS)
    gx = ops.rms_norm_backward(g, None, tt, rr, w)[0]
    assert torch.equal(x.grad, gx + gx)
    with torch.no_grad():
        assert not norm.rms_norm(x, w).requires_grad


@pytest.mark.parametrize("C", [64, 257])
def test_gradients_against_differences(C):
    rows = 9
    x, r, g, gt, w = _inputs(rows, C, F32, F32)
    y, total, rstd = ops.add_rms_norm(x, r, w, EPS)
    gx, gw = (_np(t) for t in ops.rms_norm_backward(g, gt, total, rstd, w))
    rng = np.random.default_rng(1)
    dx, dw = (rng.standard_normal(s) for s in ((rows, C), C))
    f = lambda t: ((_np(g) * R.rms_norm_fwd(_np(total) + t * dx, _np(w) + t * dw, EPS)[0]).sum()  # noqa: E731
                   + (_np(gt) * (_np(total) + t * dx)).sum())
    diff = (f(1e-5) - f(-1e-5)) / 2e-5
    got = (gx * dx).sum() + (gw * dw).sum()
    # f32 gradients (2^-24 x the chains above, at most 80) and the differences' own 1e-10 x third derivatives
    lim = 80 * U * (np.abs(gx * dx).sum() + np.abs(gw * dw).sum()) + 1e-6 * max(1.0, abs(diff))
    assert abs(got - diff) <= lim


def test_repeats_graphs_streams_and_workspaces():
    """The same bits again, from a captured graph, from another stream and beside a second graph."""
    shapes = [(300, 1024, BF), (40, 1023, F32), (1500, 77, HF)]
    for rows, C, dt in shapes:
        x, r, g, gt, w = _inputs(rows, C, dt, F32)

        def step():
            y, total, rstd = ops.add_rms_norm(x, r, w, EPS)
            return (y, total, rstd, *ops.rms_norm_backward(g, gt, total, rstd, w), *ops.add_rms_norm_int8(x, r, w, EPS))

        want = step()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
            graphs.append((graph, out))
        side = torch.cuda.Stream()
        for _ in range(3):
            for graph, _ in graphs:
                graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            alone = step()
        side.synchronize()
        for out in (alone, *(o for _, o in graphs), step()):
            assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_matches_torch():
    x, _, g, _, w = _inputs(300, 1000, F32, F32)
    xs, ws = (t.clone().requires_grad_() for t in (x, w))
    nn.functional.rms_norm(xs, (1000,), ws, EPS).backward(g)
    xo, wo = (t.clone().requires_grad_() for t in (x, w))
    norm.rms_norm(xo, wo, EPS).backward(g)
    for a, b in ((xo, xs), (wo, ws)):
        torch.testing.assert_close(a.grad, b.grad, atol=2e-4, rtol=2e-5)


def test_refusals():
    x, r, g, gt, w = _inputs(4, 64, BF, BF)
    rstd = ops.rms_norm(x, w, EPS)[1]
    refused = [
        lambda: ops.rms_norm(x, w.cpu(), EPS),
        lambda: ops.rms_norm(x, w, -1.0),
        lambda: ops.rms_norm_int8(x, w, float("nan")),
        lambda: ops.add_rms_norm(x, r.cpu(), w, EPS),
        lambda: ops.add_rms_norm(x, r[:1], w, EPS),
        lambda: ops.rms_norm_backward(g, gt.cpu(), x, rstd, w),
        lambda: ops.rms_norm_backward(g, None, x, rstd.cpu(), w),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            ops.rms_norm(dual, w, EPS)


@pytest.mark.parametrize("C", [2048, 2047])
def test_offsets_past_32_bits(C):
    """More than 2^31 values: the last rows against a call on them alone."""
    rows, last = 1_100_000, 64
    g = torch.Generator(device="cuda").manual_seed(C)
    x = torch.empty(rows, C, device="cuda", dtype=BF).normal_(generator=g)
    w = torch.rand(C, device="cuda", generator=g)
    y, total, rstd = ops.add_rms_norm(x, x, w, EPS)
    few = ops.add_rms_norm(x[-last:].clone(), x[-last:].clone(), w, EPS)
    for a, b in zip((y, total, rstd), few):
        assert torch.equal(a[-last:], b)
    gx, gw = ops.rms_norm_backward(y, total, x, rstd, w)
    few = ops.rms_norm_backward(y[-last:].clone(), total[-last:].clone(), x[-last:].clone(), rstd[-last:].clone(), w)
    assert torch.equal(gx[-last:], few[0]) and torch.isfinite(gw).all()
    codes, scales = ops.rms_norm_int8(x, w, EPS)
    few = ops.rms_norm_int8(x[-last:].clone(), w, EPS)
    assert torch.equal(codes[-last:], few[0]) and torch.equal(scales[-last:], few[1])
