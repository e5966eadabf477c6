"""8-bit checkpoints and layer norm without a GPU: fakes, refusals before any launch, the CPU paths."""

from __future__ import annotations

import ctypes

import pytest
import torch
import torch.nn as nn

from flash_mhc import MHCLiteBlock, _native, act8, norm

ops = torch.ops.flash_mhc
BF, F32, U8 = torch.bfloat16, torch.float32, torch.uint8
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _shapes(ts):
    return [(tuple(t.shape), t.dtype) for t in (ts if isinstance(ts, (tuple, list)) else (ts,))]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_fakes_give_the_shapes_and_types_of_the_cuda_ops(fmt):
    from torch._subclasses.fake_tensor import FakeTensorMode

    T, n, C, nb, ct = 6, 4, 72, 3, CODES[fmt]
    with FakeTensorMode():
        x, lo = torch.empty(T, n, C, dtype=BF), torch.empty(T, C, dtype=BF)
        h, H = torch.empty(T, n), torch.empty(T, n, n)
        xc, xs = torch.empty(T, n, C, dtype=ct), torch.empty(T, n, nb, dtype=U8)
        lc, ls = torch.empty(T, C, dtype=ct), torch.empty(T, nb, dtype=U8)
        W, g32, a = torch.empty(32, n * C, dtype=BF), torch.empty(T, 32, dtype=BF), torch.empty(1)
        kept_x, kept_lo = [((T, n, C), ct), ((T, n, nb), U8)], [((T, C), ct), ((T, nb), U8)]
        assert _shapes(ops.act_quantize(x, fmt)) == kept_x
        assert _shapes(ops.act_dequantize(xc, xs, torch.float16)) == [((T, n, C), torch.float16)]
        assert _shapes(ops.fused_pre_map_q8(x, h, fmt)) == [((T, C), BF), *kept_x]
        assert _shapes(ops.fused_post_res_q8(x, lo, H, h, fmt)) == [((T, n, C), BF), *kept_lo]
        assert _shapes(ops.mhc_pre_forward_q8(x, W, a, a, a, torch.empty(32), torch.empty(24, 16), fmt)) == [
            ((T, C), BF), ((T, 32), BF), ((T,), F32), ((T, 4), F32), ((T, 4), F32), ((T, 4, 4), F32), *kept_x]
        assert _shapes(ops.pre_map_grad_h_q8(lo, xc, xs)) == [((T, n), F32)]
        assert _shapes(ops.post_res_grad_params_q8(x, xc, xs, lc, ls, h)) == [
            ((T, C), BF), ((T, n, n), F32), ((T, n), F32)]
        assert _shapes(ops.fused_rmsnorm_project_backward_q8(g32, xc, xs, W, g32, h[:, 0])) == [
            ((T, n, C), BF), ((32, n * C), BF)]
        w = torch.empty(C)
        assert _shapes(ops.layer_norm(lo, w, w, 1e-5)) == [((T, C), BF), ((T,), F32), ((T,), F32)]
        assert _shapes(ops.layer_norm_q8(lo, w, None, 1e-5, fmt)) == [
            ((T, C), BF), ((T,), F32), ((T,), F32), *kept_lo]
        st = torch.empty(T)
        assert _shapes(ops.layer_norm_backward(lo, lo, st, st, w, None)) == [
            ((T, C), BF), ((C,), F32), ((0,), F32)]
        assert _shapes(ops.layer_norm_backward_q8(lo, lc, ls, st, st, None, w)) == [
            ((T, C), BF), ((0,), F32), ((C,), F32)]


def test_ops_raise_on_cpu_tensors():
    x = torch.zeros(4, 4, 32, dtype=BF)
    with pytest.raises(NotImplementedError):
        act8.quantize(x)
    with pytest.raises(NotImplementedError):
        norm.layer_norm(x)


def _status(name, *args):
    L = _native.lib()
    return getattr(L, name)(*args), L.fmhc_last_error().decode()


def test_c_abi_refuses_bad_arguments_before_any_launch():
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(257)  # never dereferenced
    quant = lambda x=p, dt=1, c=p, f=0, s=p, rows=4, C=64: _status(  # noqa: E731
        "fmhc_act_quantize", x, dt, c, f, s, rows, C, None)
    assert quant(rows=-1)[0] == 1 and quant(C=0)[0] == 1 and quant(C=(1 << 28) + 1)[0] == 1
    assert quant(dt=3) == (2, quant(dt=3)[1]) and "element type" in quant(dt=3)[1]
    assert quant(f=2)[0] == 2 and quant(x=None)[0] == 1 and quant(s=None)[0] == 1
    assert quant(x=odd)[0] == 3
    assert quant(x=None, c=None, s=None, rows=0) == (0, "")
    assert _status("fmhc_act_dequantize", p, 0, None, p, 1, 4, 64, None)[0] == 1
    assert _status("fmhc_act_dequantize", p, -1, p, p, 1, 4, 64, None)[0] == 2

    k3 = lambda h=p, f=0, n=4: _status("fmhc_k3_fwd_q8", p, h, p, p, p, f, 8, n, 64, None)  # noqa: E731
    assert k3(n=3)[0] == 1 and k3(f=5)[0] == 2 and k3(h=ctypes.c_void_p(264))[0] == 3
    assert _status("fmhc_k4_fwd_q8", p, p, p, p, p, None, p, 0, 8, 4, 64, None)[0] == 1
    assert _status("fmhc_k3_bwd_q8", p, p, p, 0, None, 8, 4, 64, None)[0] == 1
    assert _status("fmhc_k4_bwd_q8", p, p, p, p, p, 9, p, p, p, p, 8, 4, 64, None)[0] == 2
    assert _status("fmhc_k4_bwd_q8", p, p, p, p, p, 0, p, p, p, p, -8, 4, 64, None)[0] == 1

    size = _native.lib().fmhc_k1_bwd_q8_workspace_size
    assert size(0, 64) == 0 and size(8, 64) > 0 and size(8, 64) % 256 == 0
    k1 = lambda ws=p, b=1 << 40, x=p, gw=p: _status(  # noqa: E731
        "fmhc_k1_bwd_q8", p, x, p, 0, p, p, p, p, gw, ws, b, 8, 4, 64, None)
    assert k1(b=size(8, 64) - 1)[0] == 6 and k1(ws=ctypes.c_void_p(128))[0] == 3
    assert k1(x=None)[0] == 1 and k1(gw=None)[0] == 1


def test_c_abi_refuses_bad_layer_norm_arguments():
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(258)
    fwd = lambda x=p, dt=1, w=p, pdt=0, eps=1e-5, c=None, f=0, s=None, rows=4, C=64: _status(  # noqa: E731
        "fmhc_layer_norm_fwd", x, dt, w, p, pdt, eps, p, p, p, c, f, s, rows, C, None)
    assert fwd(dt=7)[0] == 2 and fwd(pdt=-1)[0] == 2 and fwd(x=None)[0] == 1
    assert fwd(eps=-1.0)[0] == 1 and fwd(eps=float("nan"))[0] == 1
    assert fwd(c=p)[0] == 1 and fwd(c=p, s=p, f=4)[0] == 2
    assert fwd(w=odd)[0] == 3 and fwd(C=0)[0] == 1 and fwd(rows=-2)[0] == 1
    assert fwd(x=None, rows=0) == (0, "")

    size = _native.lib().fmhc_layer_norm_bwd_workspace_size
    assert size(0, 64) == 0 and size(5, 0) == 0 and size(5, 64) % 256 == 0 and size(5, 64) > 0
    bwd = lambda x=p, c=None, s=None, gw=p, ws=p, b=1 << 40: _status(  # noqa: E731
        "fmhc_layer_norm_bwd", p, 1, x, c, 0, s, p, p, p, 0, p, gw, p, ws, b, 4, 64, None)
    assert bwd(x=None)[0] == 1 and bwd(c=p, s=p)[0] == 1 and bwd(c=p)[0] == 1
    assert bwd(gw=odd)[0] == 3 and bwd(ws=None)[0] == 1 and bwd(b=size(4, 64) - 1)[0] == 6
    assert bwd(ws=ctypes.c_void_p(128))[0] == 3


def test_layer_norm_module_is_torchs_on_cpu():
    torch.manual_seed(0)
    ours, ref = norm.LayerNorm(24, checkpoint_format="int8"), nn.LayerNorm(24)
    assert {k: v.shape for k, v in ours.state_dict().items()} == {k: v.shape for k, v in ref.state_dict().items()}
    x = torch.randn(3, 5, 24)
    assert torch.equal(ours(x), ref(x))
    assert list(norm.LayerNorm(24, bias=False).state_dict()) == ["weight"]
    assert list(norm.LayerNorm(24, elementwise_affine=False).state_dict()) == []
    with pytest.raises(ValueError, match="last dimension"):
        ours(torch.randn(3, 23))
    with pytest.raises(ValueError, match="format"):
        norm.LayerNorm(24, checkpoint_format="int4")


def test_block_argument_and_cpu_path():
    with pytest.raises(ValueError, match="checkpoint_format"):
        MHCLiteBlock(4, 16, nn.Identity(), checkpoint_format="fp8")
    torch.manual_seed(0)
    layer = nn.Linear(16, 16)
    plain, kept = MHCLiteBlock(4, 16, layer), MHCLiteBlock(4, 16, layer, checkpoint_format="int8")
    kept.load_state_dict(plain.state_dict())
    x = torch.randn(3, 4, 16)
    assert torch.equal(plain(x), kept(x))
