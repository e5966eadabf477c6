"""Root-mean-square norm and 8-bit linear layers: their plain forms, and the cases they are measured at.

``run`` computes one pass of an operator: with ``own`` false in elementary torch
operations in 32 bits, with ``own`` true by the framework's ops.  ``exact`` is
the definition in 64 bits.

* norm: y = x rstd w with rstd = 1 / sqrt(<x^2> + eps) over the last dimension, and its gradients.
* add_norm: the same of total = x + residual, rounded to x's type; the gradient of
  total, which the layers behind hand back, joins that of the norm.
* quantize: a row in 8 bits: scale = a / 127 with a the row's largest magnitude (at
  least 2^-100), codes = x / scale rounded to nearest even; and the values that they
  stand for.  A row with an infinity or a NaN has codes 0 and the scale NaN.
* norm8: total as above, and its norm in 8 bits, not rounded in between.
* linear: y = xs ws (xc . wc) + b from 8-bit rows of activations and of a weight,
  each with its scales; the sum of products is a whole number and exact.
"""

import math
import os
import sys

import torch

own = False

EPS = 1e-6
LEAST = 2.0**-100  # smallest magnitude that a row's scale is made for
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------- the cases


def listed():
    return [
        # A norm's training step: a handful of rows of odd width in 32 bits, and a batch in bf16.
        {"name": "norm, 37 rows", "op": "norm", "T": 37, "C": 1023, "dtype": "f32", "params": "f32"},
        {"name": "norm, 65536 rows", "op": "norm", "T": 65536, "C": 2048, "dtype": "bf16", "params": "bf16"},
        # The same behind a residual's addition: a ragged batch with 32-bit parameters, and a large batch.
        {"name": "add and norm, 2051 rows", "op": "add_norm", "T": 2051, "C": 1000, "dtype": "f16", "params": "f32"},
        {"name": "add and norm, 131072 rows", "op": "add_norm", "T": 131072, "C": 1024, "dtype": "bf16", "params": "bf16"},
        # Activations put into 8 bits in front of a linear layer that no norm precedes: a short prompt, and a batch of prompts.
        {"name": "quantise, 193 rows", "op": "quantize", "T": 193, "C": 1000, "dtype": "f16"},
        {"name": "quantise, 32768 rows", "op": "quantize", "T": 32768, "C": 4096, "dtype": "bf16"},
        # Serving a layer's entrance: one token, and a batch of prompts.
        {"name": "add and norm to 8 bits, 1 row", "op": "norm8", "T": 1, "C": 4096, "dtype": "bf16", "params": "bf16"},
        {"name": "add and norm to 8 bits, 65536 rows", "op": "norm8", "T": 65536, "C": 2048, "dtype": "bf16", "params": "bf16"},
        # Linear layers from 8 bits: one token, an odd layer with a bias, a batch of sequences that decode, and a batch of prompts.
        {"name": "linear, 1 row", "op": "linear", "T": 1, "K": 4096, "N": 4096, "out": "bf16", "bias": False},
        {"name": "linear, 33 rows of odd width", "op": "linear", "T": 33, "K": 1023, "N": 1001, "out": "f32", "bias": True},
        {"name": "linear, 256 rows", "op": "linear", "T": 256, "K": 4096, "N": 16384, "out": "bf16", "bias": False},
        {"name": "linear, 16384 rows", "op": "linear", "T": 16384, "K": 4096, "N": 16384, "out": "bf16", "bias": True},
    ]


def draw(rng):
    op = rng.choice(["norm", "add_norm", "quantize", "norm8", "linear", "linear", "linear"])
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    if op == "linear":
        size = lambda: rng.choice([spread(16, 16384), -(-spread(16, 16384) // 16) * 16])  # noqa: E731
        K, N = size(), size()
        T = min(spread(1, 65536), 16384 * 4096 * 16384 // (K * N), 16384 * 16384 // N, 16384 * 16384 // K)
        return {"op": op, "T": T, "K": K, "N": N, "out": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "bias": rng.choice([True, False])}
    C = spread(8, 8192)
    C = rng.choice([C, -(-C // 8) * 8, -(-C // 32) * 32, -(-C // 32) * 32])
    case = {"op": op, "T": min(spread(1, 131072), 65536 * 1024 // C), "C": C, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op != "quantize":
        case["params"] = rng.choice([case["dtype"], "f32"])
    return case


# ------------------------------------------------------ the format, plainly


def _quantize(v):
    """Rows of f32 values -> codes and scales."""
    a = v.abs().amax(-1)
    bad = ~torch.isfinite(a)
    a = a.clamp(min=LEAST)
    q = torch.where(bad.unsqueeze(-1), 0.0, v * (127.0 / a).unsqueeze(-1)).round().clamp(-127.0, 127.0)
    return q.to(torch.int8), torch.where(bad, math.nan, a / 127.0)


def _restored(case):
    """The type that 8-bit rows are looked at in: the activations' 16-bit type."""
    return torch.float16 if case["dtype"] == "f16" else torch.bfloat16


# ------------------------------------------------------------------ prepare


def _values(g, rows, C, dtype):
    """Activations: a spread of scales over the channels and the rows, and a few channels above the rest."""
    x = torch.randn(rows, C, generator=g, device="cuda")
    x *= torch.exp(0.25 * torch.randn(C, generator=g, device="cuda"))
    x *= torch.exp(0.1 * torch.randn(rows, 1, generator=g, device="cuda"))
    far = torch.randint(0, C, (max(1, C // 256),), generator=g, device="cuda")
    x[:, far] *= 4.0
    return x.to(dtype)


def _aligned_rows(codes):
    """The same codes with rows that start at multiples of 16 bytes, as 8-bit rows are kept."""
    T, K = codes.shape
    kept = torch.empty(T, -(-K // 16) * 16, dtype=codes.dtype, device=codes.device)[:, :K]
    return kept.copy_(codes)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    s = {"case": case}
    op, T = case["op"], case["T"]
    if op == "linear":
        K, N = case["K"], case["N"]
        for name, rows in (("x", T), ("w", N)):
            v = _values(g, rows, K, torch.float32) * (1.0 if name == "x" else K**-0.5)
            codes, s[name + "s"] = _quantize(v)
            s[name + "c"] = _aligned_rows(codes)
        s["b"] = (0.1 * randn(N)).to(DTYPES[case["out"]]) if case["bias"] else None
        return s
    C, dt = case["C"], DTYPES[case["dtype"]]
    s["x"] = _values(g, T, C, dt)
    if op != "quantize":
        s["w"] = (1 + 0.2 * randn(C)).to(DTYPES[case["params"]])
    if op in ("add_norm", "norm8"):
        s["r"] = _values(g, T, C, dt)
    if op in ("norm", "add_norm"):
        s["g"] = randn(T, C).to(dt)
    if op == "add_norm":
        s["gt"] = randn(T, C).to(dt)
    return s


# ---------------------------------------------------------------------- run


def _ops():
    if "flash_mhc" not in sys.modules:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-mhc_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import flash_mhc  # noqa: F401  (registers the ops)
    return torch.ops.flash_mhc


def _run_own(s):
    ops, c = _ops(), s["case"]
    op = c["op"]
    if op == "norm":
        y, rstd = ops.rms_norm(s["x"], s["w"], EPS)
        return (y, rstd, *ops.rms_norm_backward(s["g"], None, s["x"], rstd, s["w"]))
    if op == "add_norm":
        y, total, rstd = ops.add_rms_norm(s["x"], s["r"], s["w"], EPS)
        return (y, total, rstd, *ops.rms_norm_backward(s["g"], s["gt"], total, rstd, s["w"]))
    if op == "quantize":
        codes, scales = ops.row_quantize(s["x"])
        return scales, ops.row_dequantize(codes, scales, _restored(c))
    if op == "norm8":
        codes, scales, total = ops.add_rms_norm_int8(s["x"], s["r"], s["w"], EPS)
        return scales, total, ops.row_dequantize(codes, scales, _restored(c))
    return ops.int8_linear(s["xc"], s["xs"], s["wc"], s["ws"], s["b"], DTYPES[c["out"]])


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    op = c["op"]
    if op == "linear":
        y = torch.matmul(s["xc"].float(), s["wc"].float().t()) * s["xs"][:, None] * s["ws"]
        if s["b"] is not None:
            y = y + s["b"].float()
        return y.to(DTYPES[c["out"]])
    x = s["x"].float()
    if op == "quantize":
        codes, scales = _quantize(x)
        return scales, (codes.float() * scales[:, None]).to(_restored(c))
    dt = s["x"].dtype
    if op != "norm":
        total = (x + s["r"].float()).to(dt)
        x = total.float()
    rstd = torch.rsqrt(x.square().mean(-1) + EPS)
    w = s["w"].float()
    xh = x * rstd[:, None]
    if op == "norm8":
        codes, scales = _quantize(xh * w)
        return scales, total, (codes.float() * scales[:, None]).to(_restored(c))
    g = s["g"].float()
    gw = g * w
    gx = rstd[:, None] * (gw - xh * (gw * xh).mean(-1, keepdim=True))
    g_w = (g * xh).sum(0).to(s["w"].dtype)
    y = (xh * w).to(dt)
    if op == "norm":
        return y, rstd, gx.to(dt), g_w
    return y, total, rstd, (gx + s["gt"].float()).to(dt), g_w


# --------------------------------------------------------------------- work


def work(case):
    op, T = case["op"], case["T"]
    size = lambda k: torch.finfo(DTYPES[case[k]]).bits // 8  # noqa: E731
    if op == "linear":
        K, N, o = case["K"], case["N"], size("out")
        return {"bytes": T * K + N * K + 4 * (T + N) + T * N * o + (N * o if case["bias"] else 0), "flops": 2 * T * N * K}
    C, e = case["C"], size("dtype")
    if op == "quantize":  # x in, codes and scales out and in again, 16-bit values out
        return {"bytes": T * ((e + 4) * C + 8), "flops": 4 * T * C}
    p = size("params")
    if op == "norm8":  # x, residual in, total out; codes and scales out and in again, 16-bit values out
        return {"bytes": T * ((3 * e + 4) * C + 8) + C * p, "flops": 9 * T * C}
    # Forward x in, y out; backward g, x in, grad_x out; rstd out and in; the weight twice, its gradient.
    n = 5 if op == "norm" else 8  # with a residual also: it and total, and total's gradient
    return {"bytes": T * (n * e * C + 8) + 3 * C * p, "flops": (14 if op == "norm" else 16) * T * C}


# -------------------------------------------------------------------- exact


def _exact_quantize(v):
    """The values that rows of 64-bit values stand for in 8 bits, and their scales, by division."""
    a = v.abs().max(-1).values
    scale = torch.maximum(a, torch.full_like(a, LEAST)) / 127
    return torch.round(v / scale[:, None]) * scale[:, None], scale


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        y = torch.einsum("tk,nk->tn", s["xc"].double(), s["wc"].double())
        y *= s["xs"].double()[:, None]
        y *= s["ws"].double()
        return y if s["b"] is None else y.add_(s["b"].double())
    x = s["x"].double()
    if op == "quantize":
        values, scale = _exact_quantize(x)
        return scale, values
    total = None
    if op != "norm":
        total = x + s["r"].double()
        x = total.to(s["x"].dtype).double()
    w = s["w"].double()
    C = case["C"]
    rms = torch.sqrt(torch.einsum("tc,tc->t", x, x) / C + EPS)
    y = x / rms[:, None] * w
    if op == "norm8":
        values, scale = _exact_quantize(y)
        return scale, total, values
    g = s["g"].double()
    dot = torch.einsum("tc,tc,c->t", g, x, w)
    gx = (g * w) / rms[:, None] - x * (dot / (C * rms**3))[:, None]
    g_w = torch.einsum("tc,tc,t->c", g, x, 1 / rms)
    if op == "norm":
        return y, 1 / rms, gx, g_w
    return y, total, 1 / rms, gx + s["gt"].double(), g_w
