"""GPU parity of rows in 8 bits, the 8-bit linear layer and what serves with them, against float64.

u = 2^-24.  A linear layer's sum of products is exact; what is rounded is the sum's
conversion, the product of the scales, their product with the sum and, with the
bias, the result (u each), and the output's type (half a step).
"""

from __future__ import annotations

import copy
import threading

import numpy as np
import pytest
import torch
import torch.nn as nn

from flash_mhc import MHCLiteBlock, _native, int8, norm
from oracle import rms_int8_oracle as R

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device"),
]

ops = torch.ops.flash_mhc
U = 2.0 ** -24
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, rows, C, dtype=F32):
    return (torch.randn(rows, C, generator=g, device="cuda") * torch.exp(torch.randn(rows, 1, generator=g, device="cuda"))).to(dtype)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("C", [1, 7, 8, 16, 40, 256, 264, 1000, 1023, 2048, 4096, 4104, 9000, 40000])
def test_rows_to_and_from_8_bits(C, dtype):
    for rows in (1, 3, 67, 1300) if C <= 1100 else (1, 3, 300):
        x = _rows(_gen(rows + C), rows, C, dtype)
        codes, scales = int8.quantize_rows(x)
        assert codes.stride() == (-(-C // 16) * 16, 1)
        v = x.double()
        a = v.abs().amax(-1)
        assert ((scales.double() - a / 127).abs() <= U * a / 127).all()
        q = v * (127 / a)[:, None]
        # 127 / a and the product are rounded in f32
        assert ((codes.double() - q).abs() <= 0.5 + 2 * U * q.abs()).all()
        for out in (BF, HF, F32):
            got = int8.dequantize_rows(codes, scales, out)
            want = (codes.double() * scales.double()[:, None]).float().to(out)  # the f32 product is exact to u, then rounded
            assert got.dtype == out and torch.equal(got, (codes.float() * scales[:, None]).to(out)) and got.shape == want.shape


def test_rows_that_are_not_finite_and_layouts():
    x = _rows(_gen(0), 9, 300)
    x[2, 7], x[4, 299], x[5], x[6] = float("nan"), float("-inf"), 0.0, 1e-37
    codes, scales = int8.quantize_rows(x)
    assert torch.isnan(scales[[2, 4]]).all() and not codes[[2, 4, 5, 6]].any() and torch.isfinite(scales[[0, 5, 6]]).all()
    assert torch.isnan(int8.dequantize_rows(codes, scales, F32)[[2, 4]]).all()
    wc, ws = int8.quantize_rows(_rows(_gen(1), 20, 300))
    y = int8.linear(codes, scales, wc, ws, dtype=F32)
    assert torch.isnan(y[[2, 4]]).all() and torch.isfinite(y[[0, 1, 3, 7, 8]]).all() and not y[5].any()
    base = _rows(_gen(3), 60, 400, BF)
    for v in (base[:, ::2], base.t(), base[::3], base.reshape(-1)[1:1 + 50 * 400].view(50, 400),
              base.view(3, 4, 5, 400), base[7], base[:1].expand(9, 400)):
        codes, scales = int8.quantize_rows(v)
        c2, s2 = int8.quantize_rows(v.contiguous().clone())
        assert codes.shape == v.shape and scales.shape == v.shape[:-1] and torch.equal(codes, c2) and torch.equal(scales, s2)
        assert torch.equal(int8.dequantize_rows(codes, scales), int8.dequantize_rows(codes.contiguous(), scales))
    none = int8.quantize_rows(base[:0])
    assert none[0].shape == (0, 400) and int8.dequantize_rows(*none).shape == (0, 400)


def _codes(g, rows, K):
    """Codes in longer rows whose spare bytes hold 77."""
    pad = -(-K // 16) * 16
    t = torch.full((rows, pad), 77, dtype=torch.int8, device="cuda")
    t[:, :K] = torch.randint(-127, 128, (rows, K), generator=g, device="cuda", dtype=torch.int8)
    return t[:, :K]


def _check_linear(xc, xs, wc, ws, b, out):
    y = int8.linear(xc, xs, wc, ws, b, out)
    # both sides' products are whole numbers below 2^53: this matrix product is exact
    want = (xc.double().reshape(-1, xc.shape[-1]) @ wc.double().t()).view(*xc.shape[:-1], wc.shape[0])
    want = want * (xs.double().unsqueeze(-1) * ws.double())
    lim = 3 * U * want.abs()
    if b is not None:
        want = want + b.double()
        lim = lim + U * want.abs()
    half = U if out == F32 else torch.finfo(out).eps / 2
    lim = lim + half * (want.abs() + lim) + (2.0 ** -25 if out == HF else 1e-44)
    assert y.dtype == out and y.shape == want.shape
    over = (y.double() - want).abs() - lim
    assert not torch.isnan(over).any() and over.max().item() <= 0, (over.max().item(), over.argmax().item())
    return y


def _operands(T, N, K, bias=F32, seed=0):
    g = _gen(seed + T * 7 + N * 3 + K)
    r = lambda n: torch.exp(torch.randn(n, generator=g, device="cuda")) / K ** 0.5 / 70  # noqa: E731
    b = None if bias is None else torch.randn(N, generator=g, device="cuda").to(bias)
    return _codes(g, T, K), r(T), _codes(g, N, K), r(N), b


@pytest.mark.parametrize("K", [1, 15, 16, 17, 127, 128, 129, 1000, 1023, 4096])
@pytest.mark.parametrize("T", [1, 2, 3, 7, 8, 9, 16, 17, 31, 33, 64, 65, 127, 129, 200, 256, 257])
def test_linear(T, K):
    for N, out, bias in ((1, F32, F32), (31, BF, None), (128, BF, BF), (129, HF, F32), (257, F32, None), (1001, BF, HF)):
        _check_linear(*_operands(T, N, K, bias), out)


# several tiles per block, many steps of K, few tiles with a long K, a wide and a tall one
@pytest.mark.parametrize("T,N,K", [(3000, 4000, 256), (600, 700, 20000), (1, 16, 131071), (40, 130, 100000), (5000, 72, 300),
                                   (8, 30000, 640), (2, 20011, 512), (70, 9000, 2048), (1024, 4096, 4096), (300, 2500, 5000),
                                   (20000, 1100, 1008), (33, 16384, 1024), (511, 4097, 136), (12, 1000, 16384)])
def test_linear_at_larger_sizes(T, N, K):
    for out, bias in ((BF, BF), (F32, None)):
        a = _operands(T, N, K, bias)
        y = _check_linear(*a, out)
        for _ in range(2):
            assert torch.equal(y, int8.linear(*a, out))
    assert _native.check_device_error() == 0


# pairs of CTAs: rows that fill a tile badly, one column, odd columns, one byte of K, several tiles per pair
@pytest.mark.parametrize("T,N,K", [(129, 16001, 200), (300, 14501, 1), (2000, 3999, 1023), (4097, 1025, 17), (70000, 1, 64),
                                   (20001, 127, 129), (9000, 2305, 2000), (257, 20000, 128), (513, 8191, 640), (33000, 300, 40)])
def test_linear_in_pairs(T, N, K):
    for out, bias in ((F32, BF), (HF, None), (BF, F32)):
        _check_linear(*_operands(T, N, K, bias), out)
    assert _native.check_device_error() == 0


def test_linear_at_the_ends_of_the_range():
    """Every product at its largest: the sum reaches 2.1e9; and codes of -128, which quantising never gives."""
    for T in (1, 5, 40, 300):
        for K in (131071, 4096):
            for a, b in ((127, 127), (127, -127), (-128, -128)):
                xc, wc = (torch.full((n, -(-K // 16) * 16), v, dtype=torch.int8, device="cuda")[:, :K] for n, v in ((T, a), (20, b)))
                y = int8.linear(xc, torch.ones(T, device="cuda"), wc, torch.ones(20, device="cuda"), dtype=F32)
                assert (y == float(np.float32(a * b * K))).all()


def test_linear_layouts():
    g = _gen(5)
    for K in (64, 50):
        xc, xs, wc, ws, b = _operands(24, 70, K)
        want = int8.linear(xc, xs, wc, ws, b)
        wide = torch.full((24, 320), 9, dtype=torch.int8, device="cuda")
        wide[:, 32:32 + K] = xc
        odd = torch.full((24 * (K + 1) + 1,), 9, dtype=torch.int8, device="cuda")[1:].view(24, K + 1)
        odd[:, :K] = xc
        for v in (wide[:, 32:32 + K], odd[:, :K], xc.contiguous(), xc.t().contiguous().t()):
            assert torch.equal(int8.linear(v, xs, wc, ws, b), want)
            assert torch.equal(int8.linear(wc, ws, v, xs), int8.linear(wc, ws, xc, xs))
        assert torch.equal(int8.linear(xc.contiguous().view(2, 3, 4, K), xs.view(2, 3, 4), wc, ws, b), want.view(2, 3, 4, 70))
        assert torch.equal(int8.linear(xc[3], xs[3], wc, ws, b), want[3])
        spread = torch.stack([xs, xs + 1], 1)[:, 0]
        assert torch.equal(int8.linear(xc, spread, wc, torch.stack([ws, ws], 1)[:, 1], torch.stack([b, b], 1)[:, 0]), want)
        assert torch.equal(int8.linear(xc[:1].expand(24, K), xs[:1].expand(24), wc, ws, b), want[:1].expand(24, 70))
        assert int8.linear(xc[:0], xs[:0], wc, ws, b).shape == (0, 70) and int8.linear(xc, xs, wc[:0], ws[:0]).shape == (24, 0)
        for n in (1, 5, 24):  # bases that are only as aligned as rows are
            assert torch.equal(int8.linear(xc[24 - n:], xs[24 - n:], wc[1:], ws[1:], b[1:]), want[24 - n:, 1:])


def test_what_lies_around_the_output_stays():
    """The kernel writes y's elements and nothing beside them."""
    for T, N, K in ((1, 33, 64), (9, 33, 64), (40, 100, 100), (130, 257, 128), (600, 129, 256)):
        for out in (BF, F32):
            xc, xs, wc, ws, b = _operands(T, N, K)
            around = torch.full((T * N + 64,), 3.0, dtype=out, device="cuda")
            y = around[32:32 + T * N]
            s = torch.cuda.current_stream().cuda_stream
            _native.call("fmhc_int8_linear", xc.data_ptr(), xc.stride(0), xs.data_ptr(), wc.data_ptr(), wc.stride(0), ws.data_ptr(),
                         b.data_ptr(), 0, y.data_ptr(), 0 if out == F32 else 1, T, N, K, s)
            assert torch.equal(y.view(T, N), int8.linear(xc, xs, wc, ws, b, out))
            assert (around[:32] == 3).all() and (around[32 + T * N:] == 3).all()


def test_graphs_streams_and_threads():
    cases = [_operands(T, N, K, BF) for T, N, K in ((1, 4096, 1024), (20, 1000, 1000), (300, 600, 512), (1500, 3000, 256))]
    want = [int8.linear(*a) for a in cases]
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [int8.linear(*a) for a in cases]
        graphs.append((graph, out))
    for _ in range(3):
        for graph, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, out))
    found = []

    def work():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(5):
                out = [int8.linear(*a) for a in cases]
        stream.synchronize()
        found.append(all(torch.equal(a, b) for a, b in zip(want, out)))

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert found == [True] * 3 and _native.check_device_error() == 0


def test_refusals():
    xc, xs, wc, ws, b = _operands(4, 8, 64)
    refused = [
        lambda: int8.linear(xc, xs.cpu(), wc, ws),
        lambda: int8.linear(xc, xs, wc.cpu(), ws),
        lambda: int8.linear(xc, xs, wc, ws, b.cpu()),
        lambda: int8.linear(xc, xs, wc, ws, b[:4]),
        lambda: int8.linear(xc, xs, wc, ws, b, torch.float64),
        lambda: int8.linear(xc[:, :32], xs, wc, ws),
        lambda: int8.dequantize_rows(xc, xs.cpu()),
        lambda: int8.quantize_rows(xc),
        lambda: int8.linear(*(torch.zeros(s, dtype=d, device="cuda") for s, d in (((1, 1 << 17), torch.int8), ((1,), F32)) * 2)),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("C,wide", [(256, 520), (1000, 300)])
def test_a_layer_served_in_8_bits(C, wide):
    """Norm, linear, activation, linear inside a block: each part against float64 on the part's own input, the whole
    against its parts, from a graph, and near the layer that it was made from."""
    torch.manual_seed(0)
    layer = nn.Sequential(norm.RMSNorm(C), nn.Linear(C, wide), nn.GELU(), nn.Linear(wide, C, bias=False))
    blk = MHCLiteBlock(4, C, layer).cuda().to(BF).eval()
    served = int8.convert_linears(copy.deepcopy(blk))
    assert type(served.W_all) is nn.Linear and served.layer[0].weight_scales.dtype == F32
    for T in (1, 37, 700):
        x = torch.randn(T, 4, C, device="cuda", dtype=BF)
        with torch.no_grad():
            y = served(x)
            first = served.layer[0]
            li, _, _, _, h_post, H = ops.mhc_pre_forward(x, blk.W_all.weight, blk.alpha_pre, blk.alpha_post, blk.alpha_res,
                                                         blk.W_all.bias, blk.perm_mat)
            codes, scales = int8.rms_norm_int8(li, layer[0].weight, layer[0].eps)
            mid = _check_linear(codes, scales, first.weight_codes, first.weight_scales, first.bias, BF)
            assert torch.equal(first(li), mid)
            last = served.layer[2]
            act = nn.functional.gelu(mid)
            lo = _check_linear(*int8.quantize_rows(act), last.weight_codes, last.weight_scales, None, BF)
            assert torch.equal(y, ops.fused_post_res(x, lo, H, h_post))
            # 8-bit rounding of two layers' operands: half a code each, 1/254 of a row's largest, adds up like noise
            full = blk(x)
            assert (y - full).float().norm() <= 0.02 * full.float().norm()
            graph = torch.cuda.CUDAGraph()
            static = x.clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                served(static)
            torch.cuda.current_stream().wait_stream(side)
            with torch.cuda.graph(graph):
                out = served(static)
            static.copy_(torch.randn_like(x))
            graph.replay()
            assert torch.equal(out, served(static))


def test_int8_linear_module_on_cuda():
    torch.manual_seed(0)
    lin = nn.Linear(200, 90).cuda()
    q = int8.Int8Linear.from_linear(lin, norm.RMSNorm(200, device="cuda"))
    assert q.weight_codes.stride() == (208, 1)
    x, r = torch.randn(30, 200, device="cuda"), torch.randn(30, 200, device="cuda")
    with pytest.raises(RuntimeError, match="for serving"):
        q(x.clone().requires_grad_()).sum().backward()
    with torch.no_grad():
        y, total = q(x, r)
        assert torch.equal(total, x + r) and y.dtype == F32 and torch.equal(q(total), y)
        codes, scales = int8.rms_norm_int8(total, q.norm.weight)
        plain = int8.Int8Linear.from_linear(lin)
        assert torch.equal(plain((codes, scales)), y)
        moved = copy.deepcopy(q).cpu()
        z, _ = moved(x.cpu(), r.cpu())
        # the CPU's norm may round a value across the middle between two codes: one code times the largest weight
        step = scales.max().item() * (q.weight_scales * 127).max().item()
        assert (z - y.cpu()).abs().max().item() <= 3 * step
        back = moved.cuda()
        assert back.weight_codes.stride() == (208, 1) and torch.equal(back(x, r)[0], y)
        assert q.half()(x.half(), r.half())[0].dtype == HF


def test_offsets_past_32_bits():
    """A weight, activations and an output of more than 2^32 bytes: the far ends against a call on them alone."""
    g = _gen(9)
    K = 65536
    wc = torch.randint(-127, 128, (66000, K), generator=g, device="cuda", dtype=torch.int8)
    ws = torch.rand(66000, generator=g, device="cuda")
    xc, xs = wc[-300:].flip(0).contiguous(), ws[-300:].flip(0).contiguous()
    for T in (1, 20, 300):
        y = int8.linear(xc[:T], xs[:T], wc, ws)
        for at in (slice(0, 200), slice(65500, 66000)):
            assert torch.equal(y[:, at], int8.linear(xc[:T], xs[:T], wc[at], ws[at]))
    y = int8.linear(wc, ws, xc[:5], xs[:5])
    assert torch.equal(y[-200:], int8.linear(wc[-200:], ws[-200:], xc[:5], xs[:5]))
    back = int8.dequantize_rows(wc, ws)
    assert torch.equal(back[-3:], int8.dequantize_rows(wc[-3:], ws[-3:]))
    again = int8.quantize_rows(back)
    assert torch.equal(again[0][-3:], int8.quantize_rows(back[-3:].clone())[0])
    del back, again, y, wc
    # an output of 5e9 elements
    wide = torch.randint(-127, 128, (70001, 32), generator=g, device="cuda", dtype=torch.int8)
    ones = torch.ones(70001, device="cuda")
    y = int8.linear(wide, ones, wide, ones)
    assert torch.equal(y[-100:, -100:], int8.linear(wide[-100:], ones[-100:], wide[-100:], ones[-100:]))
    assert torch.equal(y[35000:35010, 69990:], int8.linear(wide[35000:35010], ones[:10], wide[69990:], ones[:11]))


def test_compiled():
    """Through torch.compile's tracing (no code generation): the same values, and gradients for the norm."""
    torch.manual_seed(0)
    x, r, w = (torch.randn(*s, device="cuda", requires_grad=True) for s in ((40, 200), (40, 200), (200,)))
    f = lambda x, r, w: norm.add_rms_norm(x, r, w)  # noqa: E731
    c = torch.compile(f, backend="aot_eager", fullgraph=True)
    for fn in (f, c):
        y, total = fn(x, r, w)
        grads = torch.autograd.grad(y.square().sum() + total.sum(), (x, r, w))
        if fn is f:
            want = (y, total, *grads)
        else:
            assert all(torch.equal(a, b) for a, b in zip(want, (y, total, *grads)))
    lin = int8.Int8Linear.from_linear(nn.Linear(200, 90).cuda(), norm.RMSNorm(200, device="cuda"))
    with torch.no_grad():
        for a, b in zip(lin(x, r), torch.compile(lin, backend="aot_eager")(x, r)):
            assert torch.equal(a, b)
