"""GPU parity of the 8-bit checkpoint ops against the float64 oracle.

Tolerances.  Codes, scales and restored values are exact.  A sum of n products
of f32 values, in any order, is off by at most n 2^-24 times the sum of the
magnitudes; the tensor cores add without rounding to nearest, so their unit is
2^-23.  A bf16 output adds half a step, 2^-8 of its value at most.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from flash_mhc import act8
from oracle import act8_oracle as A
from oracle import mhc_oracle as O

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device"),
]

ops = torch.ops.flash_mhc
FORMATS = ["int8", "e4m3"]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U24, U23, BF16_HALF = 2.0 ** -24, 2.0 ** -23, 2.0 ** -8
# ragged, odd, one block, several blocks, a last chunk of the warp, past one warp
WIDTHS = [1, 7, 8, 24, 31, 32, 33, 40, 96, 264, 1000, 1023, 1024]


def _values(rows, C, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + rows * 31 + C)
    x = torch.randn(rows, C, generator=g, device="cuda")
    x *= torch.exp(torch.randn(rows, 1, generator=g, device="cuda"))
    return x.to(dtype)


def _np(t):
    return t.detach().to(torch.float32).double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _within(name, got, want, bound):
    err = np.abs(_np(got) - want)
    assert got.shape == want.shape, name
    worst = np.max(err - bound) if err.size else 0.0
    assert worst <= 0, f"{name}: off by {err.flat[np.argmax(err - bound)]:.3g}, {worst:.3g} over the bound"


def _check_codes(x, codes, scales, fmt):
    want_c, want_s = A.quantize(_np(x), fmt)
    assert np.array_equal(_np(scales), want_s)
    assert np.array_equal(_np(codes).astype(np.float64), want_c)
    return A.restore(want_c, want_s)


# ------------------------------------------------------------ on their own


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", WIDTHS)
def test_quantize_and_dequantize_are_exact(C, dtype, fmt):
    for rows in (1, 5, 67):
        x = _values(rows, C, dtype)
        codes, scales = act8.quantize(x, fmt)
        assert codes.shape == x.shape and codes.dtype == act8.FORMATS[fmt][1]
        want = _check_codes(x, codes, scales, fmt)
        for out in DTYPES:
            got = act8.dequantize(codes, scales, out)
            ref = torch.from_numpy(want)
            if out == torch.float16:
                ref = ref.clamp(-65504, 65504)
            assert got.dtype == out and torch.equal(got.cpu(), ref.float().to(out))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("C", [40, 64, 77])
def test_quantize_edges(C, fmt):
    x = _values(9, C)
    x[0] = 0.0
    x[1, 3] = float("inf")
    x[2, C - 1] = float("nan")
    x[3, 0] = torch.finfo(torch.float32).max
    x[4] = 0.0
    x[4, 1] = 2.0 ** -149  # smallest f32
    x[5, 2] = -torch.finfo(torch.float32).max
    x[6] = 127.0 * 2.0 ** -20  # exactly M 2^k: no larger scale
    x[7] = 448.0 * 2.0 ** 9
    x[8] = torch.finfo(torch.float32).tiny
    codes, scales = act8.quantize(x, fmt)
    want = _check_codes(x, codes, scales, fmt)
    got = _np(act8.dequantize(codes, scales, torch.float32))
    assert np.array_equal(got, want.astype(np.float32).astype(np.float64), equal_nan=True)
    assert np.isnan(got[1, :32]).all() and np.isnan(got[2, C - 1])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_types_largest_values_stay_finite(dtype, fmt):
    x = torch.full((2, 64), torch.finfo(dtype).max, dtype=dtype, device="cuda")
    x[1] *= -1
    back = act8.dequantize(*act8.quantize(x, fmt), dtype)
    assert torch.isfinite(back).all()
    assert ((back.float() - x.float()).abs() <= x.float().abs() * 2.0 ** -3).all()


def test_every_code_is_restored():
    c = torch.arange(-128, 128, dtype=torch.int16).to(torch.int8).cuda()
    s = torch.full((8,), 130, dtype=torch.uint8, device="cuda")
    assert torch.equal(act8.dequantize(c, s, torch.float32), c.float() * 8)
    f = torch.arange(256, dtype=torch.int16).to(torch.uint8).view(torch.float8_e4m3fn).cuda()
    got, want = act8.dequantize(f, s, torch.float32), f.float() * 8
    assert torch.equal(got.nan_to_num(1e9), want.nan_to_num(1e9))


@pytest.mark.parametrize("fmt", FORMATS)
def test_layouts_empty_tensors_and_many_dimensions(fmt):
    base = _values(48, 200, torch.bfloat16)
    views = {"every other column": base[:, ::2], "transposed": base.t(), "rows skipped": base[::3],
             "misaligned": base.reshape(-1)[1:1 + 40 * 200].view(40, 200),
             "four dimensions": base.view(2, 4, 6, 200), "one dimension": base[3],
             "no rows": base[:0], "broadcast": base[:1].expand(5, 200)}
    for name, x in views.items():
        codes, scales = act8.quantize(x, fmt)
        assert codes.shape == x.shape and scales.shape == (*x.shape[:-1], -(-x.shape[-1] // 32)), name
        if x.numel():
            want = _check_codes(x, codes, scales, fmt)
            assert np.array_equal(_np(act8.dequantize(codes, scales, torch.float32)), want), name
        else:
            assert act8.dequantize(codes, scales).shape == x.shape
    # codes that are a view at an odd address
    codes, scales = act8.quantize(base, fmt)
    flat = torch.empty(base.numel() + 3, dtype=codes.dtype, device="cuda")
    moved = flat[3:].view(torch.uint8).view(base.shape)
    moved.copy_(codes.view(torch.uint8))
    assert torch.equal(act8.dequantize(moved.view(codes.dtype), scales), act8.dequantize(codes, scales))


# ------------------------------------------------------------- the mixings


def _coefficients(T, seed=3):
    g = torch.Generator(device="cuda").manual_seed(seed + T)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return r(T, 4), r(T, 4), r(T, 4, 4)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,C", [(1, 8), (3, 40), (37, 33), (5, 264), (130, 1000), (1000, 256), (6, 1024)])
def test_mixing_forwards_give_the_bf16_ops_outputs_and_exact_codes(T, C, fmt):
    x, lo = _values(4 * T, C, torch.bfloat16).view(T, 4, C), _values(T, C, torch.bfloat16, seed=1)
    h_pre, h_post, H = _coefficients(T)
    out, xc, xs = ops.fused_pre_map_q8(x, h_pre, fmt)
    assert torch.equal(out, ops.fused_pre_map(x, h_pre))
    _check_codes(x, xc, xs, fmt)
    out, lc, ls = ops.fused_post_res_q8(x, lo, H, h_post, fmt)
    assert torch.equal(out, ops.fused_post_res(x, lo, H, h_post))
    _check_codes(lo, lc, ls, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_mixing_forward_of_non_finite_streams(fmt):
    T, C = 4, 72
    x, lo = _values(4 * T, C, torch.bfloat16).view(T, 4, C), _values(T, C, torch.bfloat16, seed=1)
    x[1, 2, 50], x[2, 0, 0], lo[3, 71] = float("nan"), float("-inf"), float("inf")
    h_pre, h_post, H = _coefficients(T)
    out, xc, xs = ops.fused_pre_map_q8(x, h_pre, fmt)
    assert torch.equal(out.nan_to_num(7.0), ops.fused_pre_map(x, h_pre).nan_to_num(7.0))
    _check_codes(x, xc, xs, fmt)
    _, lc, ls = ops.fused_post_res_q8(x, lo, H, h_post, fmt)
    _check_codes(lo, lc, ls, fmt)
    g = torch.ones(T, C, device="cuda").bfloat16()
    gh = ops.pre_map_grad_h_q8(g, xc, xs)
    assert torch.isnan(gh[1, 2]) and torch.isnan(gh[2, 0]) and int(torch.isnan(gh).sum()) == 2


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,C", [(1, 1), (1, 8), (3, 40), (37, 33), (5, 264), (130, 1000), (515, 256), (6, 1024)])
def test_mixing_backwards_from_checkpoints(T, C, fmt):
    x, lo = _values(4 * T, C, torch.bfloat16).view(T, 4, C), _values(T, C, torch.bfloat16, seed=1)
    xc, xs = act8.quantize(x, fmt)
    lc, ls = act8.quantize(lo, fmt)
    x8, lo8 = act8.dequantize(xc, xs, torch.float32), act8.dequantize(lc, ls, torch.float32)
    go, g1 = _values(4 * T, C, torch.bfloat16, seed=2).view(T, 4, C), _values(T, C, torch.bfloat16, seed=4)
    _, h_post, H = _coefficients(T)

    gh = ops.pre_map_grad_h_q8(g1, xc, xs)
    want = np.einsum("tjc,tc->tj", _np(x8), _np(g1))
    _within("grad_h_pre", gh, want, (C + 2) * U24 * O.k3_bwd_abs(_np(g1), _np(x8)) + 1e-30)

    glo, gH, ghp = ops.post_res_grad_params_q8(go, xc, xs, lc, ls, h_post)
    aH, aP = O.k4_bwd_abs(_np(go), _np(x8), _np(lo8))
    _within("grad_H", gH, np.einsum("tic,tjc->tij", _np(go), _np(x8)), (C + 2) * U24 * aH + 1e-30)
    _within("grad_h_post", ghp, np.einsum("tic,tc->ti", _np(go), _np(lo8)), (C + 2) * U24 * aP + 1e-30)
    want = np.einsum("ti,tic->tc", _np(h_post), _np(go))
    a = np.einsum("ti,tic->tc", np.abs(_np(h_post)), np.abs(_np(go)))
    _within("grad_layer_output", glo, want, BF16_HALF * np.abs(want) + 4 * U24 * a)
    # the bf16 op gives the same grad_layer_output
    assert torch.equal(glo, ops.post_res_grad_params(go, x, lo, H, h_post)[0])


# ------------------------------------------------------------ the projection


def _projection(T, C, seed=5):
    g = torch.Generator(device="cuda").manual_seed(seed + T + C)
    W = (torch.randn(32, 4 * C, generator=g, device="cuda") / (4 * C) ** 0.5).bfloat16()
    go = torch.randn(T, 32, generator=g, device="cuda").bfloat16()
    x = _values(4 * T, C, torch.bfloat16, seed).view(T, 4, C)
    proj, inv = ops.fused_rmsnorm_project(x.view(T, 4 * C), W)
    return x, W, go, proj, inv


# widths whose K1 runs on the tensor cores (C % 32 == 0) and widths whose does
# not; token counts of less than a tile, a tile and one, many tiles
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,C", [(1, 32), (7, 24), (33, 33), (129, 64), (128, 96), (300, 160), (1, 1024),
                                 (65, 1000), (1024, 256), (4100, 512), (300, 1056), (2000, 2048)])
def test_projection_backward_from_a_checkpoint(T, C, fmt):
    x, W, go, proj, inv = _projection(T, C)
    xc, xs = act8.quantize(x, fmt)
    x8 = _np(act8.dequantize(xc, xs, torch.float32)).reshape(T, 4 * C)
    gx, gW = ops.fused_rmsnorm_project_backward_q8(go, xc, xs, W, proj, inv)
    assert gx.shape == (T, 4, C) and gW.shape == (32, 4 * C)
    r, g, p, w = _np(inv), _np(go), _np(proj), _np(W)
    want = r[:, None] * (g @ w) - ((g * p).sum(1) * r * r / (4 * C))[:, None] * x8
    a = r[:, None] * (np.abs(g) @ np.abs(w)) + (np.abs(g * p).sum(1) * r * r / (4 * C))[:, None] * np.abs(x8)
    _within("grad_x", gx.reshape(T, 4 * C), want, BF16_HALF * np.abs(want) + 40 * U23 * a + 1e-30)
    gos = _np((go.float() * inv[:, None]).bfloat16())
    want = gos.T @ x8
    _within("grad_W", gW, want, BF16_HALF * np.abs(want) + (T + 8) * U23 * (np.abs(gos).T @ np.abs(x8)) + 1e-30)


def test_projection_backward_of_views_at_odd_addresses_and_of_non_finite_streams():
    T, C = 200, 64
    x, W, go, proj, inv = _projection(T, C)
    xc, xs = act8.quantize(x)
    want = ops.fused_rmsnorm_project_backward_q8(go, xc, xs, W, proj, inv)

    def moved(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        v = flat[1:].view(t.shape)
        v.copy_(t)
        return v

    got = ops.fused_rmsnorm_project_backward_q8(*(moved(t) for t in (go, xc, xs, W, proj, inv)))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # a block of a checkpoint that stands for NaN reaches exactly its columns
    bad = xs.clone()
    bad[17, 2, 1] = 255
    gx, gW = ops.fused_rmsnorm_project_backward_q8(go, xc, bad, W, proj, inv)
    nan = torch.zeros(T, 4, C, dtype=torch.bool, device="cuda")
    nan[17, 2, 32:] = True
    assert torch.equal(torch.isnan(gx), nan) and torch.equal(gx[~nan], want[0][~nan])
    assert torch.equal(torch.isnan(gW).all(0), nan[17].reshape(-1)) and not torch.isnan(gW[:, ~nan[17].reshape(-1)]).any()


@pytest.mark.parametrize("fmt", FORMATS)
def test_projection_backward_against_differences(fmt):
    """d/dt <g, project(x + t dx, W + t dW)> at t = 0, for x that a checkpoint holds exactly."""
    T, C = 40, 64
    x = act8.dequantize(*act8.quantize(_values(4 * T, C, torch.bfloat16), fmt)).view(T, 4, C)
    xc, xs = act8.quantize(x, fmt)
    assert torch.equal(act8.dequantize(xc, xs), x)
    _, W, go, _, _ = _projection(T, C)
    proj, inv = ops.fused_rmsnorm_project(x.view(T, 4 * C), W)
    gx, gW = ops.fused_rmsnorm_project_backward_q8(go, xc, xs, W, proj, inv)
    rng = np.random.default_rng(0)
    xd, wd = rng.standard_normal((T, 4 * C)), rng.standard_normal((32, 4 * C)) / (4 * C) ** 0.5
    f = lambda t: (_np(go) * np.asarray(_project(_np(x).reshape(T, -1) + t * xd, _np(W) + t * wd))).sum()  # noqa: E731
    diff = (f(1e-4) - f(-1e-4)) / 2e-4
    got = (_np(gx).reshape(T, -1) * xd).sum() + (_np(gW) * wd).sum()
    # each gradient is off by 2^-8 of itself for its own rounding, and grad_x
    # by 2^-8 more for the bf16 proj in its formula, grad_W for the bf16 g/rms
    lim = 2 * BF16_HALF * (np.linalg.norm(_np(gx)) * np.linalg.norm(xd)
                           + np.linalg.norm(_np(gW)) * np.linalg.norm(wd))
    assert abs(got - diff) <= lim


def _project(x, W):
    return (x @ W.T) / np.sqrt((x * x).mean(1) + 1e-6)[:, None]


# ----------------------------------------------------------------- refusals


def test_refusals():
    T, C = 4, 64
    x, lo = _values(4 * T, C, torch.bfloat16).view(T, 4, C), _values(T, C, torch.bfloat16)
    h_pre, h_post, H = _coefficients(T)
    xc, xs = act8.quantize(x)
    lc, ls = act8.quantize(lo)
    e4, _ = act8.quantize(lo, "e4m3")
    g32, W, inv = torch.zeros(T, 32, device="cuda").bfloat16(), torch.zeros(32, 4 * C, device="cuda").bfloat16(), h_pre[:, 0]
    refused = [
        lambda: act8.quantize(x, "int4"),
        lambda: act8.quantize(x.double()),
        lambda: act8.quantize(x[..., :0]),
        lambda: act8.quantize(torch.zeros((), device="cuda")),
        lambda: act8.dequantize(xc, xs[..., :1]),
        lambda: act8.dequantize(xc, xs.float()),
        lambda: act8.dequantize(xc, xs.cpu()),
        lambda: act8.dequantize(xc.to(torch.int16), xs),
        lambda: act8.dequantize(xc, xs, torch.float64),
        lambda: ops.fused_pre_map_q8(x[:, :3], h_pre[:, :3], "int8"),
        lambda: ops.fused_pre_map_q8(x, h_pre[:3], "int8"),
        lambda: ops.fused_pre_map_q8(x, h_pre.cpu(), "int8"),
        lambda: ops.fused_pre_map_q8(x.float(), h_pre, "int8"),
        lambda: ops.fused_post_res_q8(x, lo[:, :32], H, h_post, "int8"),
        lambda: ops.fused_post_res_q8(x, lo, H[:, :3], h_post, "int8"),
        lambda: ops.fused_post_res_q8(x, lo, H, h_post.cpu(), "int8"),
        lambda: ops.pre_map_grad_h_q8(lo[:3], xc, xs),
        lambda: ops.pre_map_grad_h_q8(lo, xc, xs[:, :, :1]),
        lambda: ops.post_res_grad_params_q8(x, xc, xs, e4, ls, h_post),
        lambda: ops.post_res_grad_params_q8(x, xc, xs, lc[:3], ls[:3], h_post),
        lambda: ops.post_res_grad_params_q8(x, xc, xs.cpu(), lc, ls, h_post),
        lambda: ops.fused_rmsnorm_project_backward_q8(g32[:, :16], xc, xs, W, g32, inv),
        lambda: ops.fused_rmsnorm_project_backward_q8(g32, xc, xs, W[:, :64], g32, inv),
        lambda: ops.fused_rmsnorm_project_backward_q8(g32, xc, xs, W, g32, inv[:2]),
        lambda: ops.fused_rmsnorm_project_backward_q8(g32, xc, xs, W.cpu(), g32, inv),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_empty_batch():
    x = torch.empty(0, 4, 64, device="cuda").bfloat16()
    lo = torch.empty(0, 64, device="cuda").bfloat16()
    h, H = torch.empty(0, 4, device="cuda"), torch.empty(0, 4, 4, device="cuda")
    _, xc, xs = ops.fused_pre_map_q8(x, h, "int8")
    _, lc, ls = ops.fused_post_res_q8(x, lo, H, h, "int8")
    assert ops.pre_map_grad_h_q8(lo, xc, xs).shape == (0, 4)
    assert ops.post_res_grad_params_q8(x, xc, xs, lc, ls, h)[1].shape == (0, 4, 4)
    g32 = torch.empty(0, 32, device="cuda").bfloat16()
    W = torch.randn(32, 256, device="cuda").bfloat16()
    gx, gW = ops.fused_rmsnorm_project_backward_q8(g32, xc, xs, W, g32, h[:, 0])
    assert gx.shape == (0, 4, 64) and not gW.any()
