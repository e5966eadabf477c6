"""CPU oracle (numpy, float64) of the 8-bit activation checkpoints and the layer norm.

The format and the formulas are those stated in include/flashmhc.h; nothing
here shares code with the kernels.
"""

from __future__ import annotations

import numpy as np

BLOCK = 32
MOST = {"int8": 127.0, "e4m3": 448.0}
TOP_SCALE = {"int8": 248, "e4m3": 246}


def _blocks(x):
    x = np.asarray(x, dtype=np.float64)
    pad = -x.shape[-1] % BLOCK
    x = np.concatenate([x, np.zeros((*x.shape[:-1], pad))], axis=-1)
    return x.reshape(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK)


def e4m3_round(q):
    """Nearest e4m3 value (ties to even) of |q| <= 448, as float64."""
    q = np.asarray(q, dtype=np.float64)
    _, k = np.frexp(q)  # |q| = m 2^k, 1/2 <= m < 1: exponent k - 1, at least -6
    step = np.exp2(np.maximum(k - 1, -6) - 3.0)
    return np.rint(q / step) * step


def quantize(x, fmt: str):
    """(code values as float64, scale bytes) of x (..., C)."""
    C = np.asarray(x).shape[-1]
    v = _blocks(x)
    bad = ~np.isfinite(v).all(axis=-1)
    v = np.where(bad[..., None], 0.0, v)
    a = np.abs(v).max(axis=-1)
    e = np.zeros(a.shape, dtype=np.int64)
    for k in range(TOP_SCALE[fmt]):  # the smallest byte with a <= M 2^(e - 127)
        e += a > MOST[fmt] * 2.0 ** (k - 127)
    q = np.clip(v * np.exp2(127.0 - e)[..., None], -MOST[fmt], MOST[fmt])
    q = np.rint(q) if fmt == "int8" else e4m3_round(q)
    q = q.reshape(*q.shape[:-2], -1)[..., :C]
    return q, np.where(bad, 255, e).astype(np.uint8)


def restore(codes, scales):
    """float64 values that (code values, scale bytes) stand for."""
    codes = np.asarray(codes, dtype=np.float64)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127.0))
    return codes * np.repeat(s, BLOCK, axis=-1)[..., : codes.shape[-1]]


def layer_norm_fwd(x, weight, bias, eps: float):
    """y, mean, rstd in float64; weight and bias may be None."""
    x = np.asarray(x, dtype=np.float64)
    mean = x.mean(axis=-1)
    rstd = 1.0 / np.sqrt(np.square(x - mean[..., None]).mean(axis=-1) + eps)
    y = (x - mean[..., None]) * rstd[..., None]
    if weight is not None:
        y = y * np.asarray(weight, dtype=np.float64)
    if bias is not None:
        y = y + np.asarray(bias, dtype=np.float64)
    return y, mean, rstd


def layer_norm_bwd(g, x, mean, rstd, weight):
    """grad_x, grad_weight, grad_bias in float64, and the sums of magnitudes that
    bound their rounding errors: (scale of grad_x, sum |g xh|, sum |g|)."""
    g, x, mean, rstd = (np.asarray(a, dtype=np.float64) for a in (g, x, mean, rstd))
    C = x.shape[-1]
    xh = (x - mean[..., None]) * rstd[..., None]
    gw = g if weight is None else g * np.asarray(weight, dtype=np.float64)
    c1 = gw.mean(axis=-1, keepdims=True)
    c2 = (gw * xh).mean(axis=-1, keepdims=True)
    gx = rstd[..., None] * (gw - c1 - xh * c2)
    a1 = np.abs(gw).mean(axis=-1, keepdims=True)
    a2 = np.abs(gw * xh).mean(axis=-1, keepdims=True)
    scale = np.abs(rstd[..., None]) * (np.abs(gw) + a1 + np.abs(xh) * a2)
    rows = lambda a: a.reshape(-1, C).sum(axis=0)  # noqa: E731
    return (gx, rows(g * xh), rows(g)), (scale, rows(np.abs(g * xh)), rows(np.abs(g)))
