"""The 8-bit linear layer's waits that give up, on a GPU and without a fault: a lost copy is reported, what was not
computed is NaN, everything else is as without it, and later calls run as before."""

from __future__ import annotations

import time

import pytest
import torch

from flash_mhc import _native, int8

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device"),
]


# pairs of CTAs, one CTA per tile, clusters of four that split K; (rows, columns) of y that the lost copy costs
@pytest.mark.parametrize("T,N,K,lost", [(1024, 4096, 2048, None), (64, 1000, 1024, (32, 128)), (16, 1024, 4096, (16, 128))])
def test_a_lost_copy_is_reported(T, N, K, lost):
    g = torch.Generator(device="cuda").manual_seed(T)
    xc, wc = (torch.randint(-127, 128, (n, K), generator=g, device="cuda", dtype=torch.int8) for n in (T, N))
    xs, ws = torch.rand(T, generator=g, device="cuda"), torch.rand(N, generator=g, device="cuda")
    assert _native.check_device_error() == 0
    want = int8.linear(xc, xs, wc, ws)
    y = torch.zeros_like(want)
    t0 = time.monotonic()
    _native.call("fmhc_debug_int8_linear_lost_copy", xc.data_ptr(), K, xs.data_ptr(), wc.data_ptr(), K, ws.data_ptr(),
                 y.data_ptr(), T, N, K, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()  # returns: every wait is bounded
    assert time.monotonic() - t0 < 30.0
    code = _native.check_device_error()
    assert 0x201 <= code <= 0x215, hex(code)
    assert _native.check_device_error() == 0  # read and cleared
    gone = torch.isnan(y)
    assert gone.any() and torch.equal(y[~gone], want[~gone])
    if lost is not None:
        assert gone[: lost[0], : lost[1]].all() and gone.sum().item() == lost[0] * lost[1]
    assert torch.equal(int8.linear(xc, xs, wc, ws), want)
    assert _native.check_device_error() == 0
