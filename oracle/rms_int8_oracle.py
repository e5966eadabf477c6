"""CPU oracle (numpy, float64) of the root-mean-square norm, rows in 8 bits and linear layers from them.

The format and the formulas are those stated in include/flashmhc.h; nothing
here shares code with the kernels.
"""

from __future__ import annotations

import numpy as np

LEAST = 2.0 ** -100


def _f64(a):
    return None if a is None else np.asarray(a, dtype=np.float64)


def rms_norm_fwd(v, weight, eps: float):
    """y, rstd in float64; weight may be None."""
    v, weight = _f64(v), _f64(weight)
    rstd = 1.0 / np.sqrt(np.square(v).mean(axis=-1) + eps)
    y = v * rstd[..., None]
    return (y if weight is None else y * weight), rstd


def rms_norm_bwd(g, grad_total, v, rstd, weight):
    """grad_v, grad_weight in float64, and the magnitudes that bound their rounding
    errors: (terms of grad_v, sum |g xh|)."""
    g, v, rstd, weight, gt = _f64(g), _f64(v), _f64(rstd), _f64(weight), _f64(grad_total)
    C = v.shape[-1]
    xh = v * rstd[..., None]
    gw = g if weight is None else g * weight
    dot = (gw * xh).mean(axis=-1, keepdims=True)
    gx = rstd[..., None] * (gw - xh * dot)
    size = rstd[..., None] * (np.abs(gw) + np.abs(xh) * np.abs(gw * xh).mean(axis=-1, keepdims=True))
    if gt is not None:
        gx, size = gx + gt, size + np.abs(gt)
    rows = lambda a: a.reshape(-1, C).sum(axis=0)  # noqa: E731
    return (gx, rows(g * xh)), (size, rows(np.abs(g * xh)))


def row_scales(v):
    """Scale of each row; NaN for rows that are not finite."""
    v = _f64(v)
    bad = ~np.isfinite(v).all(axis=-1)
    a = np.abs(np.where(bad[..., None], 0.0, v)).max(axis=-1)
    return np.where(bad, np.nan, np.maximum(a, LEAST) / 127.0)


def row_quotients(v):
    """v / scale before rounding: codes are the nearest whole numbers.  0 in rows that are not finite."""
    s = row_scales(v)
    with np.errstate(invalid="ignore"):
        return np.where(np.isnan(s)[..., None], 0.0, _f64(v) / s[..., None])


def linear(codes, scales, weight_codes, weight_scales, bias):
    """y in float64 and |y| without its bias."""
    acc = _f64(codes) @ _f64(weight_codes).T
    y = acc * (_f64(scales)[..., None] * _f64(weight_scales))
    return (y if bias is None else y + _f64(bias)), np.abs(y)
