"""Rows of any width: every place in a word that a row can start at, every number of lanes, warps and rows that
share a block, and what lies beside a row in memory.

u = 2^-24; tolerances as in test_gpu_rms_norm.py: sums of a row in chains of at most D = 45 + C / 256 additions,
of a column in at most rows + 16, half a step for a 16-bit output, half a code and the relative error for a code.
"""

from __future__ import annotations

import os
import subprocess
import sys

import pytest
import torch

from flash_mhc import _native, int8

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device"),
]

ops = torch.ops.flash_mhc
U = 2.0 ** -24
EPS = 1e-6
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
# all residues of 8 at one to sixteen chunks; both sides of a warp, two chunks per lane and teams of warps
WIDTHS = [*range(1, 26), 31, 33, 57, 63, 64, 65, 71, 72, 119, 121, 127, 128, 129, 131, 135, 241, 249, 255, 257, 263,
          505, 509, 513, 515, 519, 761, 1017, 1025, 1029, 2041, 2049, 3001, 4093, 6001, 8170, 8178, 8179, 8185]


def _inputs(rows, C, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 31 + C)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return (*((r(rows, C) * torch.exp(0.5 * r(rows, 1))).to(dtype) for _ in range(4)), 1 + 0.3 * r(C))


def _half(dtype, v):
    if dtype == F32:
        return 2 * U * v.abs()
    return torch.finfo(dtype).eps / 2 * v.abs() + (2.0 ** -25 if dtype == HF else 0.0)


def _near(name, got, want, lim):
    over = (got.double() - want).abs() - lim
    assert got.shape == want.shape and not torch.isnan(over).any() and over.max().item() <= 0, (name, over.max().item())


def _check_all(x, r, g, gt, w, rows=None):
    """All ops on these rows; only those in ``rows`` are compared (the others hold what is not finite)."""
    C, dt = x.shape[-1], x.dtype
    rel = (0.5 * (53 + C / 256) + 8) * U
    at = slice(None) if rows is None else rows
    total = x + r
    y, t, rstd = ops.add_rms_norm(x, r, w, EPS)
    codes, scales, t2 = ops.add_rms_norm_int8(x, r, w, EPS)
    assert torch.equal(t[at], total[at]) and torch.equal(t2[at], total[at])
    y1, rstd1 = ops.rms_norm(total, w, EPS)
    codes1, scales1 = ops.rms_norm_int8(total, w, EPS)
    for a, b in ((y, y1), (rstd, rstd1), (codes, codes1), (scales, scales1)):
        assert torch.equal(a[at], b[at])
    v = total.double()
    rs = 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)
    want = v * rs * w.double()
    _near("rstd", rstd[at], rs[at, 0], rel * rs[at, 0])
    _near("y", y[at], want[at], (rel * want.abs() + _half(dt, want) * (1 + rel) + 1e-37)[at])
    s = want.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100) / 127
    _near("scales", scales[at], s[at, 0], (rel + 2 * U) * s[at, 0])
    q = want / s
    _near("codes", codes[at], q[at], (0.5 + (2 * rel + 4 * U) * q.abs())[at])
    c, s = ops.row_quantize(x)
    a = x.double().abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    _near("row scales", s[at], (a / 127)[at, 0], U * (a / 127)[at, 0])
    q = x.double() * 127 / a
    _near("row codes", c[at], q[at], (0.5 + 2 * U * q.abs())[at])
    for out in (dt, F32):
        assert torch.equal(ops.row_dequantize(c, s, out)[at], (c.float() * s[:, None]).to(out)[at])
    for up in (None, gt):
        gx, gw = ops.rms_norm_backward(g, up, total, rstd, w)
        gd, rd = g.double(), rstd.double()[:, None]
        xh = v * rd
        dot = (gd * w.double() * xh).mean(-1, keepdim=True)
        gx_want = rd * (gd * w.double() - xh * dot)
        size = rd * ((gd * w.double()).abs() + xh.abs() * (gd * w.double() * xh).abs().mean(-1, keepdim=True))
        if up is not None:
            gx_want, size = gx_want + up.double(), size + up.double().abs()
        off = (45 + C / 256 + 16) * U * size
        _near("grad_x", gx[at], gx_want[at], (off + _half(dt, gx_want.abs() + off) + 1e-30)[at])
        if rows is None:
            terms = (gd * xh).abs().sum(0)
            _near("grad_w", gw, (gd * xh).sum(0), (x.shape[0] + 16) * U * terms + 2 * U * (gd * xh).sum(0).abs() + 1e-30)
    assert torch.equal(ops.rms_norm(total, None, EPS)[0][at], ops.rms_norm(total, torch.ones_like(w), EPS)[0][at])


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("C", WIDTHS)
def test_every_width(C, dtype):
    for rows in (1, 2, 9, 150, 1201) if C < 600 else (1, 9, 150, 601):
        _check_all(*_inputs(rows, C, dtype))


@pytest.mark.parametrize("C", [1, 3, 8, 13, 40, 77, 100, 127, 300, 511, 770, 1023, 2500])
def test_many_rows(C):
    """Several rows after one another in every group of lanes, in numbers that are no multiple of what fits."""
    for rows in (148 * 24 - 1, 148 * 24 + 1, 148 * 100 + 7, 60013):
        if rows * C < 4e7:
            _check_all(*_inputs(rows, C, BF))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("C", [5, 77, 127, 300, 1023, 1025])
def test_a_row_does_not_see_its_neighbours(C, dtype):
    """NaN and infinities in every other row: chunks of memory are shared by two rows."""
    for first in (0, 1):
        x, r, g, gt, w = _inputs(301, C, dtype, seed=first)
        x[first::2], r[first::4], g[first::2], gt[first::2] = float("nan"), float("inf"), float("inf"), float("nan")
        _check_all(x, r, g, gt, w, slice(1 - first, None, 2))
        codes, scales = ops.row_quantize(x)
        assert torch.isnan(scales[first::2]).all() and not codes[first::2].any()
        codes, scales = ops.rms_norm_int8(x, w, EPS)
        assert torch.isnan(scales[first::2]).all() and not codes[first::2].any()
        assert torch.isnan(ops.rms_norm(x, w, EPS)[0][first::2]).all()


@pytest.mark.parametrize("C", [1, 7, 9, 77, 120, 129, 515, 1023, 2049, 4093])
def test_what_lies_around_the_outputs_stays(C):
    """Spare bytes of rows of codes and what is in front of and behind every output keep their values."""
    stream = torch.cuda.current_stream().cuda_stream
    call = _native.call
    for rows in (1, 67, 500):
        for stride in (-(-C // 8) * 8, -(-C // 16) * 16 + 16):
            x, r, g, gt, w = _inputs(rows, C, BF)
            pad = 64

            def around(n, dtype, value):
                t = torch.full((n + 2 * pad,), value, dtype=dtype, device="cuda")
                return t, t[pad:pad + n]

            y_all, y = around(rows * C, BF, 3.0)
            t_all, t = around(rows * C, BF, 3.0)
            gx_all, gx = around(rows * C, BF, 3.0)
            s_all, s = around(rows, F32, 3.0)
            gw_all, gw = around(C, F32, 3.0)
            c_all, c = around(rows * stride, torch.int8, 77)
            p = lambda u: u.data_ptr()  # noqa: E731
            call("fmhc_rms_norm_fwd", p(x), 1, p(r), p(w), 0, EPS, p(y), p(t), p(s), rows, C, stream)
            n = _native.lib().fmhc_rms_norm_bwd_workspace_size(rows, C)
            ws_all, ws = around(n, torch.uint8, 9)
            ws_all = torch.full((n + 512,), 9, dtype=torch.uint8, device="cuda")
            ws = ws_all[(-p(ws_all)) % 256:][:n]
            call("fmhc_rms_norm_bwd", p(g), 1, p(gt), p(t), p(s), p(w), 0, p(gx), p(gw), p(ws), n, rows, C, stream)
            call("fmhc_rms_norm_fwd_int8", p(x), 1, p(r), p(w), 0, EPS, p(c), stride, p(s), p(t), rows, C, stream)
            codes = c.view(rows, stride)
            assert (codes[:, C:] == 77).all() and torch.equal(codes[:, :C], ops.add_rms_norm_int8(x, r, w, EPS)[0])
            c.fill_(77)
            call("fmhc_row_quantize", p(x), 1, p(c), stride, p(s), rows, C, stream)
            assert (codes[:, C:] == 77).all() and torch.equal(codes[:, :C], ops.row_quantize(x)[0])
            call("fmhc_row_dequantize", p(c), stride, p(s), p(y), 1, rows, C, stream)
            assert torch.equal(y.view(rows, C), int8.dequantize_rows(*int8.quantize_rows(x)))
            for whole, value in ((y_all, 3.0), (t_all, 3.0), (gx_all, 3.0), (s_all, 3.0), (gw_all, 3.0), (c_all, 77)):
                assert (whole[:pad] == value).all() and (whole[-pad:] == value).all()
            assert (ws_all[: (-p(ws_all)) % 256] == 9).all() and (ws_all[(-p(ws_all)) % 256 + n:] == 9).all()


CHAIN = """
import sys, torch
sys.path[:0] = [{root!r}, {root!r} + "/flash-mhc_b200"]
import flash_mhc
from flash_mhc import int8
ops = torch.ops.flash_mhc
out = []
for T, C, N in ((1, 1024, 512), (9, 1023, 300), (130, 256, 1000), (700, 2048, 700), (1500, 77, 2000)):
    g = torch.Generator(device="cuda").manual_seed(T)
    x, r = (torch.randn(T, C, generator=g, device="cuda").bfloat16() for _ in range(2))
    w, W = torch.rand(C, generator=g, device="cuda"), torch.randn(N, C, generator=g, device="cuda").bfloat16()
    wc, ws = int8.quantize_rows(W)
    for _ in range(20):
        codes, scales, total = int8.add_rms_norm_int8(x, r, w)
        y = int8.linear(codes, scales, wc, ws)
        z, rstd = ops.rms_norm(total, w, 1e-6)
        gx, gw = ops.rms_norm_backward(z, total, total, rstd, w)
        back = int8.dequantize_rows(codes, scales)
        x = (0.5 * x + 0.1 * gx.clamp(-1, 1) + 0.1 * back).clamp(-4, 4)
    out += [t.double().sum().item() for t in (y, gx, gw, back, x)] + [t.double().square().sum().item() for t in (y, gx, gw, back, x)]
print(out)
"""


def test_dependent_launches_change_no_bit():
    """A chain of the ops in which each reads what the one before wrote, with and without early launches."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    found = [subprocess.run([sys.executable, "-c", CHAIN.format(root=root)], env={**os.environ, "FLASH_MHC_PDL": v},
                            capture_output=True, text=True, timeout=300, check=True).stdout for v in "01"]
    assert found[0] == found[1] and "nan" not in found[0]
