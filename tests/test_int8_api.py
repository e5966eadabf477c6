"""Root-mean-square norm and 8-bit linear layers without a GPU: fakes, refusals before any launch, autograd, the CPU paths."""

from __future__ import annotations

import copy
import ctypes
import io

import numpy as np
import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode

from flash_mhc import MHCLiteBlock, _native, int8, norm
from oracle import rms_int8_oracle as R

ops = torch.ops.flash_mhc
BF, HF, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def _described(ts):
    return [(tuple(t.shape), t.dtype, t.stride()) for t in (ts if isinstance(ts, (tuple, list)) else (ts,))]


@pytest.mark.parametrize("C", [1, 16, 40, 72])
def test_fakes(C):
    """Shapes, types and strides: dense, but rows of codes start at multiples of 16 bytes."""
    pad = -(-C // 16) * 16
    with FakeTensorMode():
        x, w = torch.empty(C, 5, 3, dtype=BF).permute(2, 1, 0), torch.empty(C)
        full, rows = ((3, 5, C), BF, (5 * C, C, 1)), ((3, 5), F32, (5, 1))
        codes = ((3, 5, C), I8, (5 * pad, pad, 1))
        assert _described(ops.rms_norm(x, w, 1e-6)) == [full, rows]
        assert _described(ops.add_rms_norm(x, x, None, 1e-6)) == [full, full, rows]
        r = torch.empty(5, 3).t()
        assert _described(ops.rms_norm_backward(x, None, x, r, w)) == [full, ((C,), F32, (1,))]
        assert _described(ops.rms_norm_backward(x, x, x, r, None)) == [full, ((0,), F32, (1,))]
        assert _described(ops.row_quantize(x)) == [codes, rows]
        assert _described(ops.rms_norm_int8(x, w, 1e-6)) == [codes, rows]
        assert _described(ops.add_rms_norm_int8(x, x, w, 1e-6)) == [codes, rows, full]
        c, s = ops.row_quantize(x)
        assert _described(ops.row_dequantize(c, s, HF)) == [((3, 5, C), HF, (5 * C, C, 1))]
        wc, ws = ops.row_quantize(torch.empty(7, C))
        assert _described(ops.int8_linear(c, s, wc, ws, None, BF)) == [((3, 5, 7), BF, (35, 7, 1))]
        assert _described(ops.int8_linear(c[0, 0], s[0, 0], wc, ws, w, F32)) == [((7,), F32, (1,))]


def test_ops_raise_on_cpu_tensors():
    x = torch.zeros(4, 32, dtype=BF)
    for call in (lambda: norm.rms_norm(x), lambda: norm.add_rms_norm(x, x), lambda: int8.quantize_rows(x),
                 lambda: int8.rms_norm_int8(x), lambda: int8.add_rms_norm_int8(x, x),
                 lambda: int8.linear(x.to(I8), torch.zeros(4), x.to(I8), torch.zeros(4))):
        with pytest.raises(NotImplementedError):
            call()


def _status(name, *args):
    L = _native.lib()
    return getattr(L, name)(*args), L.fmhc_last_error().decode()


def test_c_abi_refuses_bad_arguments_before_any_launch():
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(257)  # never dereferenced
    fwd = lambda x=p, dt=1, r=None, w=p, pdt=0, eps=1e-6, y=p, t=None, s=p, rows=4, C=64: _status(  # noqa: E731
        "fmhc_rms_norm_fwd", x, dt, r, w, pdt, eps, y, t, s, rows, C, None)
    assert fwd(dt=3)[0] == 2 and fwd(pdt=-1)[0] == 2 and fwd(x=None)[0] == 1 and fwd(y=None)[0] == 1
    assert fwd(eps=-1.0)[0] == 1 and fwd(eps=float("nan"))[0] == 1 and fwd(rows=-1)[0] == 1 and fwd(C=0)[0] == 1
    assert fwd(r=p)[0] == 1 and fwd(t=p)[0] == 1 and "go together" in fwd(t=p)[1]
    assert fwd(x=odd)[0] == 3 and fwd(w=odd)[0] == 3 and fwd(s=odd)[0] == 3 and fwd(r=odd, t=p)[0] == 3
    assert fwd(x=None, rows=0) == (0, "")
    q = lambda c=p, st=64, s=p, rows=4: _status(  # noqa: E731
        "fmhc_rms_norm_fwd_int8", p, 1, None, p, 0, 1e-6, c, st, s, None, rows, 64, None)
    assert q(st=63)[0] == 1 and "apart" in q(st=63)[1] and q(c=None)[0] == 1 and q(s=None)[0] == 1 and q(s=odd)[0] == 3
    assert q(c=None, rows=0) == (0, "")
    size = _native.lib().fmhc_rms_norm_bwd_workspace_size
    assert size(0, 64) == 0 and size(5, 0) == 0 and size(5, 64) > 0 and size(5, 64) % 256 == 0
    bwd = lambda g=p, x=p, gw=p, ws=p, b=1 << 40, gt=None: _status(  # noqa: E731
        "fmhc_rms_norm_bwd", g, 1, gt, x, p, p, 0, p, gw, ws, b, 4, 64, None)
    assert bwd(g=None)[0] == 1 and bwd(x=None)[0] == 1 and bwd(ws=None)[0] == 1 and bwd(gw=odd)[0] == 3
    assert bwd(ws=ctypes.c_void_p(128))[0] == 3 and bwd(b=size(4, 64) - 1)[0] == 6 and bwd(gt=odd)[0] == 3

    assert _status("fmhc_row_quantize", p, 5, p, 64, p, 4, 64, None)[0] == 2
    assert _status("fmhc_row_quantize", p, 1, p, 60, p, 4, 64, None)[0] == 1
    assert _status("fmhc_row_quantize", p, 1, None, 64, p, 4, 64, None)[0] == 1
    assert _status("fmhc_row_quantize", odd, 1, p, 64, p, 4, 64, None)[0] == 3
    assert _status("fmhc_row_dequantize", p, 64, None, p, 1, 4, 64, None)[0] == 1
    assert _status("fmhc_row_dequantize", p, 64, p, odd, 1, 4, 64, None)[0] == 3
    assert _status("fmhc_row_dequantize", None, 64, None, None, 1, 0, 64, None) == (0, "")

    lin = lambda c=p, cs=64, s=p, w=p, wst=64, ws=p, b=None, bdt=0, y=p, ydt=1, T=4, N=8, K=64: _status(  # noqa: E731
        "fmhc_int8_linear", c, cs, s, w, wst, ws, b, bdt, y, ydt, T, N, K, None)
    assert lin(T=-1)[0] == 1 and lin(N=1 << 31)[0] == 1 and lin(K=0)[0] == 1 and lin(K=1 << 17, cs=1 << 17, wst=1 << 17)[0] == 1
    assert lin(cs=48)[0] == 1 and lin(wst=48)[0] == 1 and lin(cs=72)[0] == 3 and lin(wst=65)[0] == 3
    assert lin(bdt=9)[0] == 2 and lin(ydt=3)[0] == 2 and lin(c=None)[0] == 1 and lin(y=None)[0] == 1
    assert lin(c=ctypes.c_void_p(264))[0] == 3 and lin(w=ctypes.c_void_p(264))[0] == 3
    assert lin(b=odd)[0] == 3 and lin(y=odd)[0] == 3 and lin(s=odd)[0] == 3
    assert lin(c=None, T=0) == (0, "") and lin(y=None, N=0) == (0, "")


def test_codes_that_are_not_laid_out_are_copied():
    c = torch.arange(60, dtype=I8).view(5, 12)
    laid = int8._laid_out(c)
    assert torch.equal(laid, c) and laid.stride() == (16, 1) and int8._laid_out(laid) is laid
    for v in (c.t(), c[:, 2:7], c[:1].expand(4, 12), laid[:, 1:], c[::2], c.view(5, 3, 4)):
        t = int8._laid_out(v)
        assert torch.equal(t, v.reshape(-1, v.shape[-1]))
        assert t.data_ptr() % 16 == 0 and t.stride(1) == 1 and int8._stride(t) % 16 == 0
    wide = torch.zeros(6, 64, dtype=I8)
    assert int8._laid_out(wide[::2, :40]).data_ptr() == wide.data_ptr() and int8._stride(wide[::2, :40]) == 128


def test_what_the_ops_refuse():
    """Checks that come before any launch, on the functions that take CUDA tensors."""
    x, w, c, s = torch.zeros(4, 32, dtype=BF), torch.ones(32), torch.zeros(4, 32, dtype=I8), torch.ones(4)
    refused = [
        lambda: norm._rms_norm_cuda(x.double(), w, 1e-6),
        lambda: norm._rms_norm_cuda(x[:, :0], None, 1e-6),
        lambda: norm._rms_norm_cuda(x, w[:8], 1e-6),
        lambda: norm._rms_norm_cuda(x, w.double(), 1e-6),
        lambda: norm._rms_norm_cuda(torch.zeros((), dtype=BF), None, 1e-6),
        lambda: norm._add_rms_norm_cuda(x, x[:2], w, 1e-6),
        lambda: norm._add_rms_norm_cuda(x, x.float(), w, 1e-6),
        lambda: norm._rms_norm_backward_cuda(x, None, x[:2], s, w),
        lambda: norm._rms_norm_backward_cuda(x, None, x.float(), s, w),
        lambda: norm._rms_norm_backward_cuda(x, x[:3], x, s, w),
        lambda: norm._rms_norm_backward_cuda(x, x.float(), x, s, w),
        lambda: norm._rms_norm_backward_cuda(x, None, x, s[:2], w),
        lambda: norm._rms_norm_backward_cuda(x, None, x, s.double(), w),
        lambda: int8._row_quantize_cuda(c),
        lambda: int8._add_rms_norm_int8_cuda(x, x[:, :8], w, 1e-6),
        lambda: int8._row_dequantize_cuda(c, s, torch.int8),
        lambda: int8._row_dequantize_cuda(c, s[:2], BF),
        lambda: int8._row_dequantize_cuda(c, s.double(), BF),
        lambda: int8._row_dequantize_cuda(c.to(torch.uint8), s, BF),
        lambda: int8._int8_linear_cuda(c, s, c, s, None, torch.float64),
        lambda: int8._int8_linear_cuda(c, s, c[:, :16], s, None, BF),
        lambda: int8._int8_linear_cuda(c, s, c[0], s, None, BF),
        lambda: int8._int8_linear_cuda(c, s, c, s[:3], None, BF),
        lambda: int8._int8_linear_cuda(c, s, c, s, w, BF),
        lambda: int8._int8_linear_cuda(c, s, c, s, s.double(), BF),
        lambda: int8._int8_linear_cuda(c.float(), s, c, s, None, BF),
        lambda: int8._int8_linear_cuda(c[:, :0], s, c[:, :0], s, None, BF),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_autograd_with_fakes():
    """What requires a gradient, and that a backward through an 8-bit op raises."""
    with FakeTensorMode():
        x, r, w = (torch.empty(*s, requires_grad=True) for s in ((6, 32), (6, 32), (32,)))
        y, rstd = ops.rms_norm(x, w, 1e-6)
        assert y.requires_grad and not rstd.requires_grad
        y.sum().backward()
        assert x.grad.shape == x.shape and w.grad.shape == w.shape
        y, total, rstd = ops.add_rms_norm(x, r, w, 1e-6)
        assert y.requires_grad and total.requires_grad and not rstd.requires_grad
        x.grad = w.grad = None
        total.sum().backward()  # nothing through the norm
        assert x.grad is not None and r.grad is not None and w.grad is None
        (gx,) = torch.autograd.grad(ops.rms_norm(x, w, 1e-6)[0].sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="rms_norm has no second derivative"):
            gx.sum().backward()
        c, s = ops.row_quantize(x)
        assert not c.requires_grad and not s.requires_grad
        b = torch.empty(6, requires_grad=True)
        for name, outs in (("rms_norm_int8", ops.rms_norm_int8(x, w, 1e-6)),
                           ("add_rms_norm_int8", ops.add_rms_norm_int8(x, r, w, 1e-6)),
                           ("int8_linear", [ops.int8_linear(c, s, c, s, b, F32)])):
            for t in outs:
                if t.is_floating_point():
                    with pytest.raises(RuntimeError, match=f"{name} has no derivative"):
                        t.sum().backward(retain_graph=True)
        assert not ops.int8_linear(c, s, c, s, None, BF).requires_grad


def test_rms_norm_module_is_torchs_on_cpu():
    torch.manual_seed(0)
    ours, ref = norm.RMSNorm(24), nn.RMSNorm(24, eps=1e-6)
    assert {k: v.shape for k, v in ours.state_dict().items()} == {k: v.shape for k, v in ref.state_dict().items()}
    x, r = torch.randn(3, 5, 24), torch.randn(3, 5, 24)
    assert torch.equal(ours(x), ref(x))
    y, total = ours(x, r)
    assert torch.equal(total, x + r) and torch.equal(y, ref(x + r))
    assert list(norm.RMSNorm(24, elementwise_affine=False).state_dict()) == []
    with pytest.raises(ValueError, match="last dimension"):
        ours(torch.randn(3, 23))


def _model(C=24, wide=40):
    torch.manual_seed(0)
    return nn.Sequential(norm.RMSNorm(C), nn.Linear(C, wide), nn.GELU(), nn.Linear(wide, C, bias=False))


def _quantisation_bound(x, layer):
    """|error| of a linear layer in 8 bits: half a code of each x times |w|, half a code of each w times |x|, and both."""
    v, w = x.detach().double().numpy(), layer.weight.detach().double().numpy()
    ex, ew = R.row_scales(v)[..., None] / 2, R.row_scales(w)[:, None] / 2
    return np.abs(ex) * np.abs(w).sum(-1) + np.abs(v) @ np.abs(np.broadcast_to(ew, w.shape)).T + ex * ew[:, 0] * w.shape[1]


def test_int8_linear_on_cpu():
    torch.manual_seed(0)
    layer = nn.Linear(40, 9)
    q = int8.Int8Linear.from_linear(layer)
    x = torch.randn(2, 7, 40)
    c, s = int8._quantize_plain(x)
    want, size = R.linear(c.numpy(), s.numpy(), q.weight_codes.numpy(), q.weight_scales.numpy(), layer.bias.detach().numpy())
    with torch.no_grad():
        y = q(x)
        assert np.abs(y.numpy() - want).max() <= 4 * 2.0 ** -24 * (size + np.abs(want)).max()
        assert (np.abs(y.numpy() - layer(x).numpy()) <= 1.001 * _quantisation_bound(x, layer)).all()
        assert q((c, s)).dtype == F32 and torch.equal(q((c, s)), y)
    y = q(x.requires_grad_())
    assert y.requires_grad
    with pytest.raises(RuntimeError, match="for serving"):
        y.sum().backward()
    with pytest.raises(ValueError, match="has none"):
        q(x, x)
    with pytest.raises(ValueError, match="norm must be"):
        int8.Int8Linear(8, 8, norm=norm.RMSNorm(9))
    with pytest.raises(ValueError, match="in_features"):
        int8.Int8Linear(1 << 17, 1, device="meta")
    with pytest.raises(ValueError, match="residual must be"):
        int8.Int8Linear(8, 8, norm=norm.RMSNorm(8))(torch.zeros(3, 8), torch.zeros(8))
    with pytest.raises(ValueError, match="residual must be"):
        norm.RMSNorm(8)(torch.zeros(3, 8), torch.zeros(3, 8, dtype=BF))
    n = int8.Int8Linear.from_linear(layer, norm.RMSNorm(40))
    with pytest.raises(ValueError, match="without a norm"):
        n((c, s))
    y, total = n(x, x)
    assert torch.equal(total, x + x) and torch.equal(n(total), y)
    with pytest.raises(RuntimeError, match="for serving"):
        total.sum().backward()


def test_int8_linear_keeps_its_scales_and_layout():
    """Through changes of type, copies, state dicts and files."""
    q = int8.Int8Linear.from_linear(nn.Linear(40, 9, bias=False))
    scales, codes = q.weight_scales.clone(), q.weight_codes.clone()
    whole = copy.deepcopy(q)
    f = io.BytesIO()
    torch.save(q, f)
    f.seek(0)
    loaded = int8.Int8Linear(40, 9, bias=False)
    loaded.load_state_dict(q.state_dict())
    for m in (q.to(BF), q.half(), whole, whole.to(torch.device("cpu"), HF), torch.load(f, weights_only=False), loaded):
        assert torch.equal(m.weight_scales, scales) and m.weight_scales.dtype == F32
        assert torch.equal(m.weight_codes, codes) and m.weight_codes.stride() == (48, 1)
    assert q.dtype == HF and whole.dtype == HF and loaded.dtype == BF
    assert q.to("meta").weight_codes.is_meta


def test_convert_linears():
    m = _model()
    x = torch.randn(5, 24)
    with torch.no_grad():
        want = m(x)
        c = int8.convert_linears(copy.deepcopy(m))
        assert [type(l).__name__ for l in c] == ["Int8Linear", "GELU", "Int8Linear"] and c[0].norm is not None
        first = m[2](m[1](m[0](x)))
        bound = _quantisation_bound(m[0](x), m[1]) @ np.abs(m[3].weight.double().numpy()).T * 1.13  # |gelu'| < 1.13
        bound += _quantisation_bound(first, m[3]) * 1.2  # the second layer's input moves a little
        assert (np.abs((c(x) - want).numpy()) <= bound).all()

    class Twice(nn.Module):
        def __init__(self):
            super().__init__()
            self.a = nn.Linear(8, 8)
            self.b = self.a
            self.block = MHCLiteBlock(4, 8, nn.Sequential(nn.Linear(8, 8)))
            self.wide = nn.Linear(8, 8).double()
            self.hooked = nn.Linear(8, 8)
            self.hooked.register_forward_hook(lambda *a: None)
            self.attn = nn.MultiheadAttention(8, 2)

    t = Twice()
    assert int8.convert_linears(t) is t
    assert type(t.a) is int8.Int8Linear and t.a is t.b and type(t.block.layer[0]) is int8.Int8Linear
    assert type(t.block.W_all) is nn.Linear and type(t.wide) is nn.Linear and type(t.hooked) is nn.Linear
    assert isinstance(t.attn.out_proj, nn.Linear)
    assert type(int8.convert_linears(nn.Linear(8, 8))) is int8.Int8Linear
    with torch.no_grad():
        assert t.block(torch.randn(3, 4, 8)).shape == (3, 4, 8)


def test_convert_linears_keeps_a_sequentials_hooks():
    seen = []
    m = nn.Sequential(norm.RMSNorm(8), nn.Linear(8, 8))
    m.register_forward_hook(lambda *a: seen.append(1))
    c = int8.convert_linears(m)
    assert c is m and type(c[0]) is norm.RMSNorm and type(c[1]) is int8.Int8Linear and c[1].norm is None
    with torch.no_grad():
        c(torch.randn(2, 8))
    assert seen == [1]
