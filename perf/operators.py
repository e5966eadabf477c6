"""The 8-bit activation checkpoints and the layer norm: their plain forms, and the cases they are measured at.

``run`` computes one pass of an operator: with ``own`` false in elementary torch
operations in 32 bits, with ``own`` true by the framework's ops.  ``exact`` is
the definition in 64 bits.

The checkpoint format: blocks of 32 values along the last dimension (the last
block of a row may be shorter), one scale byte e per block standing for
2^(e - 127), and one code per value.  With a the largest magnitude of the
block, e is the smallest byte with a <= M 2^(e - 127), where M is 127 for int8
codes and 448 for e4m3 codes; codes are x / scale rounded to nearest even and
kept within [-M, M].  A block that holds an infinity or a NaN has e = 255 and
stands for NaN.
"""

import math
import os
import sys

import torch

own = False

BLOCK = 32
EPS_RMS = 1e-6
EPS_LN = 1e-5
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
#: largest code; bits that carry into the exponent above M's significand; M's exponent
FORMATS = {"int8": (127.0, 0x1FFFF, 6), "e4m3": (448.0, 0x1FFFFF, 8)}


# ---------------------------------------------------------------- the cases


def listed():
    return [
        # One layer's streams of a three-token batch, put away and restored: launch latency, odd width, half precision.
        {"name": "checkpoint, 3 tokens", "op": "checkpoint", "rows": 12, "C": 1000, "dtype": "f16", "fmt": "e4m3"},
        # The streams of one training batch (the kernel benchmark's shape), put away and restored.
        {"name": "checkpoint, 65536 tokens", "op": "checkpoint", "rows": 4 * 65536, "C": 1024, "dtype": "bf16", "fmt": "int8"},
        # A block's forward mixing with its checkpoints: a short ragged batch, and the benchmark's batch.
        {"name": "mix forward, 193 tokens", "op": "mix", "T": 193, "C": 1000, "fmt": "e4m3"},
        {"name": "mix forward, 65536 tokens", "op": "mix", "T": 65536, "C": 1024, "fmt": "int8"},
        # The post-mixing's gradients from the checkpoints: a small batch, and the block benchmark's batch.
        {"name": "post backward, 1024 tokens", "op": "post_bwd", "T": 1024, "C": 1024, "fmt": "int8"},
        {"name": "post backward, 65536 tokens", "op": "post_bwd", "T": 65536, "C": 2048, "fmt": "e4m3"},
        # The pre-mixing's and the projection's gradients from the checkpoint: a small batch, and the benchmark's.
        {"name": "pre backward, 2048 tokens", "op": "pre_bwd", "T": 2048, "C": 2048, "fmt": "e4m3"},
        {"name": "pre backward, 65536 tokens", "op": "pre_bwd", "T": 65536, "C": 1024, "fmt": "int8"},
        # A norm's training step: a handful of rows of odd width in 32 bits, and a batch in bf16.
        {"name": "layer norm, 37 rows", "op": "norm", "T": 37, "C": 1023, "dtype": "f32", "params": "f32"},
        {"name": "layer norm, 65536 rows", "op": "norm", "T": 65536, "C": 2048, "dtype": "bf16", "params": "bf16"},
        # The same with the input kept in 8 bits: mixed precision with 32-bit parameters, and the benchmark's batch.
        {"name": "8-bit norm, 16384 rows", "op": "norm_q8", "T": 16384, "C": 4096, "dtype": "f16", "params": "f32", "fmt": "e4m3"},
        {"name": "8-bit norm, 131072 rows", "op": "norm_q8", "T": 131072, "C": 1024, "dtype": "bf16", "params": "bf16", "fmt": "int8"},
    ]


def draw(rng):
    op = rng.choice(["checkpoint", "mix", "post_bwd", "pre_bwd", "norm", "norm_q8"])
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    C = spread(8, 4096)
    C = rng.choice([C, -(-C // 8) * 8, -(-C // 32) * 32, -(-C // 32) * 32])
    T = min(spread(1, 65536), 65536 * 1024 // C)
    case = {"op": op, "C": C}
    if op != "norm":
        case["fmt"] = rng.choice(["int8", "e4m3"])
    if op == "checkpoint":
        case["rows"] = 4 * T
    else:
        case["T"] = T
    if op in ("checkpoint", "norm", "norm_q8"):
        case["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("norm", "norm_q8"):
        case["params"] = rng.choice([case["dtype"], "f32"])
    return case


# ------------------------------------------------------ the format, plainly


def _blocks(x):
    """(..., C) -> (..., blocks, 32), short blocks filled with zeros."""
    C = x.shape[-1]
    n = -(-C // BLOCK)
    if n * BLOCK != C:
        x = torch.nn.functional.pad(x, (0, n * BLOCK - C))
    return x.unflatten(-1, (n, BLOCK))


def _quantize(x, fmt):
    most, carry, top = FORMATS[fmt]
    v = _blocks(x.float())
    amax = v.abs().amax(-1)
    e = (((amax.view(torch.int32) + carry) >> 23).clamp(max=254) - top).clamp(min=0)
    q = (v * ((254 - e) << 23).view(torch.float32).unsqueeze(-1)).clamp(-most, most)
    bad = ~torch.isfinite(amax)
    q = torch.where(bad.unsqueeze(-1), 0.0, q).flatten(-2)[..., : x.shape[-1]].contiguous()
    codes = q.round().to(torch.int8) if fmt == "int8" else q.to(torch.float8_e4m3fn)
    return codes, torch.where(bad, 255, e).to(torch.uint8)


def _restore(codes, scales):
    e = scales.to(torch.int32)
    s = torch.where(e == 0, 0x00400000, torch.where(e == 255, 0x7FC00000, e << 23)).view(torch.float32)
    return (_blocks(codes.float()) * s.unsqueeze(-1)).flatten(-2)[..., : codes.shape[-1]]


# ------------------------------------------------------------------ prepare


def _values(g, rows, C, dtype):
    """Activations: a spread of scales over the channels and the rows, and a few channels far above the rest."""
    x = torch.randn(rows, C, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(C, generator=g, device="cuda"))
    x *= torch.exp(0.3 * torch.randn(rows, 1, generator=g, device="cuda"))
    far = torch.randint(0, C, (max(1, C // 256),), generator=g, device="cuda")
    x[:, far] *= 12.0
    return x.to(dtype)


def _coefficients(g, T):
    h_pre = torch.sigmoid(torch.randn(T, 4, generator=g, device="cuda"))
    h_post = 2 * torch.sigmoid(torch.randn(T, 4, generator=g, device="cuda"))
    H = torch.softmax(torch.randn(T, 4, 4, generator=g, device="cuda"), -1) - h_post[:, :, None] * h_pre[:, None, :]
    return h_pre, h_post, H.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    op, C = case["op"], case["C"]
    if own:
        _framework()
    if op == "checkpoint":
        return {"case": case, "x": _values(g, case["rows"], C, DTYPES[case["dtype"]])}
    T = case["T"]
    if op in ("norm", "norm_q8"):
        dt, pt = DTYPES[case["dtype"]], DTYPES[case["params"]]
        return {"case": case, "x": _values(g, T, C, dt) + 0.5 * randn(C).to(dt), "g": randn(T, C).to(dt),
                "w": (1 + 0.2 * randn(C)).to(pt), "b": (0.1 * randn(C)).to(pt)}
    x = _values(g, 4 * T, C, torch.bfloat16).view(T, 4, C)
    s = {"case": case}
    if op == "mix":
        s["h_pre"], s["h_post"], s["H"] = _coefficients(g, T)
        s["x"], s["lo"] = x, _values(g, T, C, torch.bfloat16)
    elif op == "post_bwd":
        _, s["h_post"], _ = _coefficients(g, T)
        s["xc"], s["xs"] = _quantize(x, case["fmt"])
        s["lc"], s["ls"] = _quantize(_values(g, T, C, torch.bfloat16), case["fmt"])
        s["go"] = randn(T, 4, C).bfloat16()
    else:
        W = (randn(32, 4 * C) / math.sqrt(4 * C)).bfloat16()
        flat = x.view(T, 4 * C).float()
        s["inv"] = torch.rsqrt(flat.square().mean(-1) + EPS_RMS)
        s["proj"] = (flat @ W.float().t() * s["inv"][:, None]).bfloat16()
        s["W"] = W
        s["xc"], s["xs"] = _quantize(x, case["fmt"])
        s["go"] = randn(T, 32).bfloat16()
        s["g_in"] = randn(T, C).bfloat16()
    return s


# ---------------------------------------------------------------------- run


def _framework():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-mhc_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_mhc  # noqa: F401  (registers the ops)

    return torch.ops.flash_mhc


def _run_own(s):
    ops, c = torch.ops.flash_mhc, s["case"]
    op, fmt = c["op"], c.get("fmt")
    if op == "checkpoint":
        codes, scales = ops.act_quantize(s["x"], fmt)
        return codes, scales, ops.act_dequantize(codes, scales, s["x"].dtype)
    if op == "mix":
        return (*ops.fused_pre_map_q8(s["x"], s["h_pre"], fmt),
                *ops.fused_post_res_q8(s["x"], s["lo"], s["H"], s["h_post"], fmt))
    if op == "post_bwd":
        return ops.post_res_grad_params_q8(s["go"], s["xc"], s["xs"], s["lc"], s["ls"], s["h_post"])
    if op == "pre_bwd":
        return (ops.pre_map_grad_h_q8(s["g_in"], s["xc"], s["xs"]),
                *ops.fused_rmsnorm_project_backward_q8(s["go"], s["xc"], s["xs"], s["W"], s["proj"], s["inv"]))
    if op == "norm":
        y, mean, rstd = ops.layer_norm(s["x"], s["w"], s["b"], EPS_LN)
        return (y, mean, rstd, *ops.layer_norm_backward(s["g"], s["x"], mean, rstd, s["w"], s["b"]))
    y, mean, rstd, codes, scales = ops.layer_norm_q8(s["x"], s["w"], s["b"], EPS_LN, fmt)
    return (y, mean, rstd, codes, scales,
            *ops.layer_norm_backward_q8(s["g"], codes, scales, mean, rstd, s["w"], s["b"]))


def _norm_grads(g, x, mean, rstd, w, b):
    dt = g.dtype
    g = g.float()
    xh = (x - mean[:, None]) * rstd[:, None]
    gw = g * w.float()
    gx = rstd[:, None] * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    return gx.to(dt), (g * xh).sum(0).to(w.dtype), g.sum(0).to(b.dtype)


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    op, fmt = c["op"], c.get("fmt")
    if op == "checkpoint":
        codes, scales = _quantize(s["x"], fmt)
        v = _restore(codes, scales)
        if s["x"].dtype == torch.float16:
            v = v.clamp(-65504.0, 65504.0)
        return codes, scales, v.to(s["x"].dtype)
    if op == "mix":
        x, lo = s["x"].float(), s["lo"].float()
        out = (s["h_pre"][:, :, None] * x).sum(1).bfloat16()
        post = (torch.matmul(s["H"], x) + s["h_post"][:, :, None] * lo[:, None, :]).bfloat16()
        return (out, *_quantize(s["x"], fmt), post, *_quantize(s["lo"], fmt))
    if op == "post_bwd":
        x, lo, go = _restore(s["xc"], s["xs"]), _restore(s["lc"], s["ls"]), s["go"].float()
        g_lo = (s["h_post"][:, :, None] * go).sum(1).bfloat16()
        return g_lo, torch.matmul(go, x.transpose(1, 2)), (go * lo[:, None, :]).sum(-1)
    if op == "pre_bwd":
        T, C = c["T"], c["C"]
        x = _restore(s["xc"], s["xs"])
        g_h = (x * s["g_in"].float()[:, None, :]).sum(-1)
        flat, go, inv = x.reshape(T, 4 * C), s["go"].float(), s["inv"][:, None]
        k = (go * s["proj"].float()).sum(-1, keepdim=True) * inv * inv / (4 * C)
        gx = inv * (go @ s["W"].float()) - k * flat
        gW = (go * inv).bfloat16().float().t() @ flat
        return g_h, gx.bfloat16().view(T, 4, C), gW.bfloat16()
    x, w, b = s["x"].float(), s["w"], s["b"]
    mean = x.mean(-1)
    var = (x - mean[:, None]).square().mean(-1)
    rstd = torch.rsqrt(var + EPS_LN)
    y = ((x - mean[:, None]) * rstd[:, None] * w.float() + b.float()).to(s["x"].dtype)
    if op == "norm":
        return (y, mean, rstd, *_norm_grads(s["g"], x, mean, rstd, w, b))
    codes, scales = _quantize(s["x"], fmt)
    return (y, mean, rstd, codes, scales, *_norm_grads(s["g"], _restore(codes, scales), mean, rstd, w, b))


# --------------------------------------------------------------------- work


def work(case):
    op, C = case["op"], case["C"]
    nb = -(-C // BLOCK)
    size = lambda k: torch.finfo(DTYPES[case[k]]).bits // 8  # noqa: E731
    if op == "checkpoint":  # x in, codes and scales out and in again, x out
        return {"bytes": case["rows"] * (2 * size("dtype") * C + 2 * (C + nb)), "flops": 4 * case["rows"] * C}
    T = case["T"]
    if op == "mix":  # the two mixings run before and after the wrapped layer: each reads the streams
        return {"bytes": T * (8 * C + 16 + 2 * C + 4 * (C + nb) + 10 * C + 80 + 8 * C + C + nb), "flops": T * C * 48}
    if op == "post_bwd":
        return {"bytes": T * (8 * C + 5 * (C + nb) + 16 + 2 * C + 80), "flops": T * C * 48}
    if op == "pre_bwd":  # two ops with the coefficients' backward between them: each reads the checkpoint
        return {"bytes": T * (2 * C + 4 * (C + nb) + 16 + 4 * (C + nb) + 128 + 4 + 8 * C) + 2 * 32 * 4 * C * 2,
                "flops": T * C * 8 + 4 * T * 32 * 4 * C}
    e, p = size("dtype"), size("params")
    step = T * C * 5 * e + 4 * T * 4 + C * 5 * p  # x, y, g, x again, grad_x; mean and rstd out and in; the parameters
    if op == "norm_q8":  # written as codes, and read as codes in x's place
        step += T * (2 * (C + nb) - C * e)
    return {"bytes": step, "flops": T * C * 22}


# -------------------------------------------------------------------- exact


def _exact_scale(e):
    """2^(e - 127) in 64 bits, from a table (a power function may be off in its last bit)."""
    powers = torch.tensor([2.0 ** (i - 127) for i in range(255)] + [math.nan], dtype=torch.float64)
    return powers.to(e.device)[e.long()]


def _exact_quantize(x, fmt):
    """Codes and scale bytes by exponents and division in 64 bits."""
    most = FORMATS[fmt][0]
    C = x.shape[-1]
    pad = (-C) % BLOCK
    v = torch.cat([x.double(), x.new_zeros((*x.shape[:-1], pad), dtype=torch.float64)], -1)
    v = v.reshape(*x.shape[:-1], (C + pad) // BLOCK, BLOCK)
    m, k = torch.frexp(v.abs().max(-1).values)  # a = m 2^k with 1/2 <= m < 1
    m_most, k_most = math.frexp(most)
    e = k.to(torch.int64) - k_most + (m > m_most).long() + 127
    e = torch.where(m == 0, 0, e).clamp(0, 254 - FORMATS[fmt][2])
    q = v / _exact_scale(e)[..., None]
    q = q.clamp(-most, most).reshape(*x.shape[:-1], C + pad)[..., :C]
    codes = torch.round(q).to(torch.int8) if fmt == "int8" else q.float().to(torch.float8_e4m3fn)
    return codes, e.to(torch.uint8)


def _exact_restore(codes, scales):
    return codes.to(torch.float32).double() * _exact_scale(scales).repeat_interleave(BLOCK, -1)[..., : codes.shape[-1]]


def exact(case, seed):
    s = prepare(case, seed)
    op, fmt = case["op"], case.get("fmt")
    if op == "checkpoint":
        codes, scales = _exact_quantize(s["x"], fmt)
        return codes, scales, _exact_restore(codes, scales)
    if op == "mix":
        x, lo = s["x"].double(), s["lo"].double()
        out = torch.einsum("tj,tjc->tc", s["h_pre"].double(), x)
        post = torch.einsum("tij,tjc->tic", s["H"].double(), x)
        post += torch.einsum("ti,tc->tic", s["h_post"].double(), lo)
        return (out, *_exact_quantize(s["x"], fmt), post, *_exact_quantize(s["lo"], fmt))
    if op == "post_bwd":
        x, lo, go = _exact_restore(s["xc"], s["xs"]), _exact_restore(s["lc"], s["ls"]), s["go"].double()
        return (torch.einsum("ti,tic->tc", s["h_post"].double(), go), torch.einsum("tic,tjc->tij", go, x),
                torch.einsum("tic,tc->ti", go, lo))
    if op == "pre_bwd":
        T, C = case["T"], case["C"]
        x = _exact_restore(s["xc"], s["xs"])
        g_h = torch.einsum("tjc,tc->tj", x, s["g_in"].double())
        x = x.reshape(T, 4 * C)
        go, inv = s["go"].double(), s["inv"].double()
        gW = torch.einsum("td,tk->dk", (s["go"].float() * s["inv"][:, None]).bfloat16().double(), x)
        x *= -(torch.einsum("td,td->t", go, s["proj"].double()) * inv * inv / (4 * C))[:, None]
        x += inv[:, None] * torch.einsum("td,dk->tk", go, s["W"].double())
        return g_h, x.view(T, 4, C), gW
    x, w, b, g = (s[k].double() for k in ("x", "w", "b", "g"))
    var, mean = torch.var_mean(x, -1, correction=0)
    rstd = 1 / torch.sqrt(var + EPS_LN)
    y = torch.addcmul(b, (x - mean[:, None]) / torch.sqrt(var + EPS_LN)[:, None], w)
    kept = ()
    if op == "norm_q8":
        kept = _exact_quantize(s["x"], fmt)
        x = _exact_restore(*kept)
    xh = (x - mean[:, None]) * rstd[:, None]
    C = x.shape[-1]
    t = g * w
    gx = (t * C - t.sum(-1, keepdim=True) - xh * torch.einsum("tc,tc->t", t, xh)[:, None]) * (rstd / C)[:, None]
    return (y, mean, rstd, *kept, gx, torch.einsum("tc,tc->c", g, xh), g.sum(0))
