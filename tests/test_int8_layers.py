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
