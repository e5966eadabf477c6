"""8-bit layers without a GPU: the format that the torch paths write, what they load, what they convert."""

from __future__ import annotations

import copy
from collections import OrderedDict

import numpy as np
import pytest
import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensorMode

from flash_mhc import int8, norm


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_codes_without_a_gpu_are_the_formats(dtype):
    """127 / a rounded once to 32 bits, the product too: every code, those between two steps (x = a / 2) among them."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3000, 200, generator=g).to(dtype)
    x[:, 7] = x.float().abs().amax(-1).to(dtype)
    x[:, 8] = x[:, 7] / 2
    codes, scales = int8._quantize_plain(x)
    v = x.float().numpy()
    a = np.abs(v).max(-1)
    assert a.dtype == np.float32
    assert np.array_equal(scales.numpy(), a / np.float32(127))
    assert np.array_equal(codes.numpy(), np.rint(v * (np.float32(127) / a)[:, None]).astype(np.int8))


def test_codes_that_are_loaded_are_laid_out():
    """assign=True puts the state dict's own tensors in place, whose rows may be packed: a forward would copy them every time."""
    q = int8.Int8Linear.from_linear(nn.Linear(40, 9))
    x = torch.randn(4, 40)
    with torch.no_grad():
        want = q(x)
    packed = {k: v.contiguous() for k, v in q.state_dict().items()}
    assert packed["weight_codes"].stride() == (40, 1)
    far = torch.zeros(9 * 40 + 1, dtype=torch.int8)[1:].view(9, 40).copy_(packed["weight_codes"])
    for assign in (True, False):
        for codes in (packed["weight_codes"], packed["weight_codes"].t().contiguous().t(), far, q.weight_codes):
            m = int8.Int8Linear(40, 9, device="meta" if assign else None, dtype=torch.float32)
            m.load_state_dict({**packed, "weight_codes": codes}, assign=assign)
            assert m.weight_codes.stride() == (48, 1) and int8._laid_out(m.weight_codes) is m.weight_codes
            with torch.no_grad():
                assert torch.equal(m(x), want)
    m.load_state_dict(q.state_dict(), assign=True)
    assert m.weight_codes.data_ptr() == q.weight_codes.data_ptr()  # laid out: as it is
    whole = nn.Sequential(int8.Int8Linear(40, 9, device="meta"))
    whole.load_state_dict({"0." + k: v for k, v in packed.items()}, assign=True)
    assert whole[0].weight_codes.stride() == (48, 1)
    assert q.state_dict()["weight_codes"].data_ptr() == q.weight_codes.data_ptr()  # references, as torch's are
    with pytest.raises(RuntimeError, match="size mismatch"):
        q.load_state_dict({**packed, "weight_codes": packed["weight_codes"][:, :39]}, assign=True)
    with FakeTensorMode():
        f = int8.Int8Linear(40, 9)
        f.load_state_dict(int8.Int8Linear(40, 9).state_dict(), assign=True)
        assert f.weight_codes.stride() == (48, 1)


def _named():
    m = nn.Sequential(OrderedDict(n=norm.RMSNorm(8), up=nn.Linear(8, 12), drop=nn.Dropout(0.9), down=nn.Linear(12, 8)))
    m.note = ["kept"]
    return m


def test_a_container_that_gets_shorter_keeps_names_modes_and_attributes():
    m = _named()
    m.drop.eval()
    m.n.eval()
    whole = nn.Module()
    whole.ffn = m
    assert int8.convert_linears(whole) is whole
    c = whole.ffn
    assert type(c) is nn.Sequential and list(c._modules) == ["up", "drop", "down"] and c.note == ["kept"]
    assert c.training and not c.drop.training and c.up.training and c.down.training
    assert c.up.norm is m.n and not c.up.norm.training and type(c.down) is int8.Int8Linear
    assert set(c.state_dict()) == {"up.weight_codes", "up.weight_scales", "up.bias", "up.norm.weight",
                                   "down.weight_codes", "down.weight_scales", "down.bias"}
    c.register_forward_hook(lambda *a: None)
    assert list(m._modules) == ["n", "up", "drop", "down"] and not m._forward_hooks  # the longer one is as it was
    numbered = int8.convert_linears(nn.Sequential(norm.RMSNorm(8), nn.Linear(8, 8), norm.RMSNorm(8), nn.Linear(8, 8)).eval())
    assert list(numbered._modules) == ["0", "1"] and not any(t.training for t in numbered.modules())
    numbered.append(nn.GELU())
    assert list(numbered._modules) == ["0", "1", "2"]


def test_torchs_own_modules_run_converted():
    """Those that read a linear layer's weight keep it."""
    torch.manual_seed(0)
    x = torch.randn(2, 5, 8)
    enc = lambda: nn.TransformerEncoderLayer(8, 2, 16, batch_first=True)  # noqa: E731
    for m, args in ((enc(), (x,)), (nn.TransformerEncoder(enc(), 2), (x,)),
                    (nn.TransformerDecoderLayer(8, 2, 16, batch_first=True), (x, x)),
                    (nn.Transformer(8, 2, 1, 1, 16, batch_first=True), (x, x)),
                    (nn.MultiheadAttention(8, 2, batch_first=True), (x, x, x)),
                    (nn.AdaptiveLogSoftmaxWithLoss(8, 20, [5, 10]), (x.view(10, 8), torch.arange(10)))):
        for mode in (True, False):
            with torch.no_grad():
                int8.convert_linears(copy.deepcopy(m).train(mode))(*args)
    layer = enc().eval()
    with torch.no_grad():
        want = layer(x)
        assert torch.equal(int8.convert_linears(layer)(x), want)
    assert type(layer.linear1) is nn.Linear and type(layer.linear2) is nn.Linear


def test_a_layer_in_several_places_stays_one():
    lin, n1, n2 = nn.Linear(8, 8), norm.RMSNorm(8), norm.RMSNorm(8)
    with torch.no_grad():
        n2.weight.fill_(2.0)
    x = torch.randn(3, 8)

    def converted(*parts):
        m = nn.Module()
        m.parts = nn.ModuleList(parts)
        c = int8.convert_linears(copy.deepcopy(m)).parts
        with torch.no_grad():
            for a, b in zip(parts, c):
                assert (a(x) - b(x)).abs().max() < 0.2 * a(x).abs().max()  # 8 bits: far from another norm's or none
        return c, [q for q in c.modules() if type(q) is int8.Int8Linear]

    c, q = converted(nn.Sequential(n1, lin), nn.Sequential(n1, lin, nn.GELU()))  # behind one norm everywhere
    assert len(q) == 1 and q[0].norm is not None and c[0][0] is c[1][0]
    c, q = converted(nn.Sequential(n1, lin), nn.Sequential(n2, lin))  # behind two
    assert len(q) == 1 and q[0].norm is None and len(c[0]) == len(c[1]) == 2
    c, q = converted(nn.Sequential(n1, lin), lin)  # with a norm and without
    assert len(q) == 1 and q[0].norm is None and c[1] is c[0][1]
    c, q = converted(lin, nn.Sequential(nn.Identity(), n1, lin))
    assert len(q) == 1 and q[0].norm is None and c[0] is c[1][2]
    c, q = converted(nn.Sequential(n1, lin), nn.Sequential(n1, nn.Linear(8, 8)))  # one norm, two layers
    assert len(q) == 2 and q[0].norm is q[1].norm is not None
    s = nn.Sequential(n1, lin)
    c, q = converted(s, s)
    assert len(q) == 1 and c[0] is c[1] and len(c[0]) == 1
    alone = int8.convert_linears(lin)
    assert type(alone) is int8.Int8Linear and alone.norm is None


def test_float64_layers_and_activations():
    torch.manual_seed(0)
    q = int8.Int8Linear.from_linear(nn.Linear(40, 9), norm.RMSNorm(40))
    x = torch.randn(4, 40)
    with torch.no_grad():
        want = q(x)
        assert q(x.double()).dtype == torch.float64 and torch.equal(q(x.double()).float(), want)
        y = q.double()(x.double())
        assert q.weight_scales.dtype == torch.float32 and y.dtype == torch.float64
        assert torch.equal(y.float(), want)
        with pytest.raises(ValueError, match="floating-point"):
            q(torch.ones(4, 40, dtype=torch.int64))
        with pytest.raises(ValueError, match="floating-point"):
            int8.Int8Linear(40, 9)(torch.ones(4, 40, dtype=torch.int8))


def test_convert_linears_sees_a_forward_of_the_modules_own():
    """A forward that was set on a module, as wrappers do, is a hook; a compiled call is the longer container's alone."""
    seen = []

    def wrapped(m):
        old = m.forward
        m.forward = lambda *a: (seen.append(type(m)), old(*a))[1]
        return m

    x = torch.randn(3, 8)
    m = nn.Sequential(wrapped(nn.Linear(8, 8)), nn.Linear(8, 8), norm.RMSNorm(8), nn.Linear(8, 8))
    c = int8.convert_linears(m)
    assert type(c[0]) is nn.Linear and [type(t) for t in c[1:]] == [int8.Int8Linear] * 2 and c[2].norm is m[2]
    s = wrapped(nn.Sequential(norm.RMSNorm(8), nn.Linear(8, 8)))
    q = int8.convert_linears(s)
    assert q is s and type(q[0]) is norm.RMSNorm and type(q[1]) is int8.Int8Linear
    with torch.no_grad():
        c(x), q(x)
    assert seen == [nn.Linear, nn.Sequential]
    p = nn.Sequential(norm.RMSNorm(8), nn.Linear(8, 8))
    p.compile(backend="eager")
    with torch.no_grad():
        assert torch.equal(int8.convert_linears(p)(x), int8.convert_linears(copy.deepcopy(nn.Sequential(*p)))(x))
