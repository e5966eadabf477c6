"""8-bit rows and layers on a GPU where they can go wrong: values between two codes, scales at the ends of f32's range,
other types, one lost copy.  u = 2^-24."""

from __future__ import annotations

import copy

import numpy as np
import pytest
import torch
import torch.nn as nn

from flash_mhc import _native, int8, norm

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device"),
]

U = 2.0 ** -24
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("C", [64, 200, 1023, 2048, 4096, 9000])
def test_codes_are_the_formats_to_the_bit(C, dtype):
    """Those between two steps among them (x = a / 2 is 63.5 steps), in the kernels and in torch on both devices."""
    x = torch.randn(2000, C, generator=_gen(C), device="cuda").to(dtype)
    x[:, 7] = x.float().abs().amax(-1).to(dtype)
    x[:, 8] = x[:, 7] / 2
    codes, scales = int8.quantize_rows(x)
    v = x.float().cpu().numpy()
    a = np.abs(v).max(-1)
    assert np.array_equal(scales.cpu().numpy(), a / np.float32(127))
    assert np.array_equal(codes.cpu().numpy(), np.rint(v * (np.float32(127) / a)[:, None]).astype(np.int8))
    for t in (x, x.cpu()):
        c, s = int8._quantize_plain(t)
        assert torch.equal(c.to(codes.device), codes) and torch.equal(s.to(scales.device), scales)


# rows of a warp, of a team of warps, of several rows per warp, of an odd width; past the widths of the other kernels
@pytest.mark.parametrize("C", [256, 2048, 4096, 64, 1023, 9000])
@pytest.mark.parametrize("size,weight", [(1e17, 3e-27), (1e-10, 1e36)])
def test_a_norm_to_8_bits_whose_weight_is_far_from_one(C, size, weight):
    """rstd w is 3e-44 or 1e39, out of f32's range, where the normalised values and their products with w are not."""
    x = (torch.randn(40, C, generator=_gen(C), device="cuda") * size).clamp(-4 * size, 4 * size)
    w = torch.linspace(1, 2, C, device="cuda") * weight
    y = x.double() / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    a = y.abs().amax(-1)
    for codes, scales, *_ in (int8.rms_norm_int8(x, w), int8.add_rms_norm_int8(x, torch.zeros_like(x), w)):
        # the sum of squares (C u, its mean's 3 u), the square root's 2 u, two products and the division: C + 8 roundings
        rel = (C + 8) * U
        assert ((scales.double() - a / 127).abs() <= rel * a / 127).all()
        assert ((codes.double() - y * (127 / a)[:, None]).abs() <= 0.5 + 2 * 127 * rel).all()


# the kernel for a handful of rows, one CTA per tile, clusters that split K, pairs of CTAs
@pytest.mark.parametrize("T,N,K", [(1, 300, 512), (5, 300, 512), (40, 300, 512), (16, 1024, 4096), (1024, 4096, 512)])
@pytest.mark.parametrize("xs,ws", [(3e-22, 2e-21), (2e-21, 3e-22), (1e34, 1e-30), (2e36, 1e-20), (1e-25, 1e25), (1e-31, 1e29)])
def test_scales_at_the_ends_of_the_range(T, N, K, xs, ws):
    """The scales' product leaves f32's range or not: y does not, and neither does the sum times the weight's scale."""
    g = _gen(T + N)
    xc, wc = (torch.randint(-127, 128, (n, K), generator=g, device="cuda", dtype=torch.int8) for n in (T, N))
    sx, sw = (torch.linspace(1, 1.5, n, device="cuda") * s for n, s in ((T, xs), (N, ws)))
    sums = (xc.double() @ wc.double().t())
    b = torch.randn(N, generator=g, device="cuda") * float(np.float32(xs * ws * 1e4))
    for bias in (None, b):
        y = int8.linear(xc, sx, wc, sw, bias, F32).double()
        want = sums * sw.double() * sx.double()[:, None]
        lim = 3 * U * want.abs()
        if bias is not None:
            want = want + bias.double()
            lim = lim + U * want.abs()
        assert ((y - want).abs() <= lim + 2.0 ** -149).all()  # the least step of f32


@pytest.mark.parametrize("T,N,K", [(1, 300, 512), (40, 300, 512), (16, 1024, 4096), (1024, 4096, 512)])
def test_a_sum_of_zero_is_zero_under_any_scales(T, N, K):
    """Orthogonal rows of codes, with scales whose product is infinite in f32: y is the bias."""
    xc, wc = torch.zeros(T, K, dtype=torch.int8, device="cuda"), torch.zeros(N, K, dtype=torch.int8, device="cuda")
    xc[:, : K // 2], wc[:, K // 2:] = 3, 5
    b = torch.randn(N, generator=_gen(N), device="cuda")
    y = int8.linear(xc, torch.full((T,), 1e30, device="cuda"), wc, torch.full((N,), 1e30, device="cuda"), b, F32)
    assert torch.equal(y, b.expand(T, N))


@pytest.mark.parametrize("bias", [True, False])
def test_float64_as_on_the_cpu(bias):
    """A layer that was converted as a whole, and float64 activations: from 32 bits, in their type."""
    torch.manual_seed(0)
    x = torch.randn(30, 200)
    q = int8.Int8Linear.from_linear(nn.Linear(200, 90, bias=bias))
    for m in (q, copy.deepcopy(q).double()):
        with torch.no_grad():
            want = m(x.double())
            c, s = int8._quantize_plain(x)
            size = (c.double() @ m.weight_codes.double().t()).abs() * s.double()[:, None] * m.weight_scales.double()
            g = copy.deepcopy(m).cuda()
            for y in (g(x.double().cuda()), g((c.cuda(), s.cuda()))):
                # three or four roundings on each side, of the sum's part and of the result
                assert ((y.double().cpu() - want).abs() <= 8 * U * (size + want.abs())).all()
            assert g(x.double().cuda()).dtype == want.dtype == torch.float64 and g((c.cuda(), s.cuda())).dtype == m.dtype


def test_a_lost_copy_costs_a_pair_its_tile_alone():
    """Pairs of CTAs, one tile each: the first tile (256 rows and columns) is NaN, everything else as without the loss."""
    T, N, K = 1024, 4096, 2048
    g = _gen(T)
    xc, wc = (torch.randint(-127, 128, (n, K), generator=g, device="cuda", dtype=torch.int8) for n in (T, N))
    xs, ws = torch.rand(T, generator=g, device="cuda"), torch.rand(N, generator=g, device="cuda")
    want = int8.linear(xc, xs, wc, ws)
    y = torch.zeros_like(want)
    _native.call("fmhc_debug_int8_linear_lost_copy", xc.data_ptr(), K, xs.data_ptr(), wc.data_ptr(), K, ws.data_ptr(),
                 y.data_ptr(), T, N, K, torch.cuda.current_stream().cuda_stream)
    assert 0x201 <= _native.check_device_error() <= 0x205 and _native.check_device_error() == 0
    lost = torch.zeros_like(y, dtype=torch.bool)
    lost[:256, :256] = True
    assert torch.equal(torch.isnan(y), lost) and torch.equal(y[~lost], want[~lost])
