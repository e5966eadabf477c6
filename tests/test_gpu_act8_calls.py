"""Calls of the 8-bit and layer-norm ops at the edges of what they allow: second derivatives,
offsets past 32 bits, the widest rows, views at odd addresses, captured graphs."""

import threading

import pytest
import torch
import torch.nn as nn
import torch.utils.checkpoint

import flash_mhc  # noqa: F401
from flash_mhc import act8, norm
from flash_mhc.block import MHCLiteBlock

pytestmark = pytest.mark.gpu

ops = torch.ops.flash_mhc
BF = torch.bfloat16


def _randn(*shape, dtype=BF):
    return torch.randn(*shape, device="cuda", dtype=dtype)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_quantising_takes_no_part_in_autograd(fmt):
    x = _randn(4, 64).requires_grad_()
    c, s = act8.quantize(x, fmt)
    assert not c.requires_grad and not s.requires_grad and not act8.dequantize(c, s).requires_grad
    want = act8.quantize(x.detach(), fmt)
    assert torch.equal(c.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s, want[1])


@pytest.mark.parametrize("fmt", [None, "int8"])
def test_second_derivatives_of_the_norm_are_refused(fmt):
    x, w = _randn(4, 64).requires_grad_(), _randn(64).requires_grad_()
    y = norm.layer_norm(x, w, None, checkpoint_format=fmt)
    g = _randn(4, 64)
    first = torch.autograd.grad(y, (x, w), g, create_graph=True)
    plain = torch.autograd.grad(norm.layer_norm(x, w, None, checkpoint_format=fmt), (x, w), g)
    assert all(torch.equal(a, b) for a, b in zip(first, plain))
    with pytest.raises(RuntimeError, match="second derivative"):
        first[0].float().pow(2).sum().backward()
    # alone with a frozen weight and a linear loss, too
    y = norm.layer_norm(x, None, None, checkpoint_format=fmt)
    first, = torch.autograd.grad(y, x, g, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        first.float().pow(2).sum().backward()


def test_second_derivatives_of_the_block_are_refused():
    b = MHCLiteBlock(4, 64, nn.Linear(64, 64), checkpoint_format="int8").cuda().to(BF)
    x = _randn(5, 4, 64).requires_grad_()
    g, = torch.autograd.grad(b(x).float().pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().pow(2).sum().backward()


@pytest.mark.parametrize("fmt", [None, "int8"])
def test_forward_mode_derivatives_are_refused(fmt):
    x = _randn(4, 64, dtype=torch.float32)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
            norm.layer_norm(dual, None, None, checkpoint_format=fmt)
        assert torch.equal(norm.layer_norm(x), norm.layer_norm(x.clone()))


def test_threads_streams_and_torchs_own_checkpointing():
    """Two threads train at once on streams of their own; the block under torch's recomputation and with its
    saved tensors on the host: all with the bits of a plain step."""
    def make(seed):
        torch.manual_seed(seed)
        layer = nn.Sequential(norm.LayerNorm(264, checkpoint_format="int8"), nn.Linear(264, 264))
        m = MHCLiteBlock(4, 264, layer, checkpoint_format="int8").cuda().to(BF)
        return m, _randn(700, 4, 264), _randn(700, 4, 264)

    def step(m, x, g, call=lambda m, x: m(x)):
        x = x.detach().requires_grad_()
        return torch.autograd.grad(call(m, x), [x, *m.parameters()], g)

    cases = [make(1), make(2)]
    want = [step(*c) for c in cases]
    same = lambda got, ref: all(torch.equal(a, b) for a, b in zip(got, ref))  # noqa: E731
    torch.cuda.synchronize()
    good = [0, 0]

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                good[i] += same(step(*cases[i]), want[i])
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert good == [20, 20]
    recompute = lambda m, x: torch.utils.checkpoint.checkpoint(m, x, use_reentrant=False)  # noqa: E731
    assert torch.equal(step(*cases[0], recompute)[0], want[0][0])
    with torch.autograd.graph.save_on_cpu():
        assert same(step(*cases[0]), want[0])


# ------------------------------------------------------ offsets past 32 bits
# Every token's or row's result has the same bits wherever it stands, so the last ones of a long
# tensor are compared with a short call's.
C = 1024
T = (1 << 31) // (4 * C) + 37  # 4 T C values: the last ones lie past 2^31
LAST = 70


def test_long_tensors_quantise_and_restore():
    x = _randn(4 * T, C)
    c, s = act8.quantize(x)
    wc, ws = act8.quantize(x[-LAST:])
    assert torch.equal(c[-LAST:], wc) and torch.equal(s[-LAST:], ws)
    assert torch.equal(act8.dequantize(c, s)[-LAST:], act8.dequantize(wc, ws))


def test_long_tensors_mixings():
    x, lo = _randn(T, 4, C), _randn(T, C)
    h, H = torch.rand(T, 4, device="cuda"), torch.rand(T, 4, 4, device="cuda")
    out, xc, xs = ops.fused_pre_map_q8(x, h, "int8")
    want = ops.fused_pre_map_q8(x[-LAST:], h[-LAST:], "int8")
    assert all(torch.equal(a[-LAST:], b) for a, b in zip((out, xc, xs), want))
    out, lc, ls = ops.fused_post_res_q8(x, lo, H, h, "int8")
    want = ops.fused_post_res_q8(x[-LAST:], lo[-LAST:], H[-LAST:], h[-LAST:], "int8")
    assert all(torch.equal(a[-LAST:], b) for a, b in zip((out, lc, ls), want))
    got = ops.post_res_grad_params_q8(out, xc, xs, lc, ls, h)
    want = ops.post_res_grad_params_q8(*(t[-LAST:] for t in (out, xc, xs, lc, ls, h)))
    assert all(torch.equal(a[-LAST:], b) for a, b in zip(got, want))
    assert torch.equal(ops.pre_map_grad_h_q8(lo, xc, xs)[-LAST:],
                       ops.pre_map_grad_h_q8(*(t[-LAST:] for t in (lo, xc, xs))))


def test_long_tensors_projection_backward():
    xc = torch.randint(-127, 128, (T, 4, C), device="cuda", dtype=torch.int8)
    xs = torch.full((T, 4, C // 32), 120, device="cuda", dtype=torch.uint8)
    W, proj, inv = _randn(32, 4 * C), _randn(T, 32), torch.rand(T, device="cuda") + 0.5
    go = torch.zeros(T, 32, device="cuda", dtype=BF)
    go[-LAST:] = _randn(LAST, 32)
    gx, gW = ops.fused_rmsnorm_project_backward_q8(go, xc, xs, W, proj, inv)
    wx, wW = ops.fused_rmsnorm_project_backward_q8(*(t[-LAST:] for t in (go, xc, xs)), W, proj[-LAST:], inv[-LAST:])
    assert torch.equal(gx[-LAST:], wx) and not gx[:-LAST].any()
    # grad_W: zero but for the last tokens' products, which are added in f32 in two groupings (70
    # products each: 2 x 70 x 2^-24 of the sum of magnitudes) and rounded to bf16 twice, each time by
    # at most 2^-8 of the value: |R(a) - R(b)| <= |a - b| + 2^-8 |a| + 2^-8 |b|.  With |a| and |b| at most
    # |R(b)| / (1 - 2^-8) + |a - b|, the roundings are within 2^-7 (1 + 2^-7) |R(b)| + 2^-7 |a - b|,
    # and the last term is within the slack of 140 for 2 x 69 additions.
    x = act8.dequantize(xc[-LAST:], xs[-LAST:], torch.float32).view(LAST, 4 * C).double()
    g = (go[-LAST:].float() * inv[-LAST:, None]).to(BF).double()
    lim = wW.double().abs() * 2**-7 * (1 + 2**-7) + g.abs().t() @ x.abs() * (140 * 2.0**-24)
    assert ((gW.double() - wW.double()).abs() <= lim).all()


@pytest.mark.parametrize("fmt", [None, "e4m3"])
def test_long_tensors_norm(fmt):
    rows = 4 * T
    x, w, b = _randn(rows, C), _randn(C), _randn(C)
    fwd = ops.layer_norm(x, w, b, 1e-5) if fmt is None else ops.layer_norm_q8(x, w, b, 1e-5, fmt)
    want = ops.layer_norm(x[-LAST:], w, b, 1e-5) if fmt is None else ops.layer_norm_q8(x[-LAST:], w, b, 1e-5, fmt)
    for a, r in zip(fwd, want):
        assert torch.equal(a[-LAST:].view(torch.uint8), r.view(torch.uint8))
    g = torch.zeros_like(x)
    g[-1] = _randn(C)  # one row: the parameters' gradients are its alone
    kept = (x,) if fmt is None else fwd[3:]
    bwd = ops.layer_norm_backward if fmt is None else ops.layer_norm_backward_q8
    got = bwd(g, *kept, fwd[1], fwd[2], w, b)
    ref = bwd(g[-LAST:], *(t[-LAST:] for t in kept), fwd[1][-LAST:], fwd[2][-LAST:], w, b)
    assert torch.equal(got[0][-LAST:], ref[0]) and torch.equal(got[1], ref[1]) and torch.equal(got[2], ref[2])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("tokens,width", [(1, 1), (5, 3), (31, 32), (32, 64), (33, 8192), (40, 8192), (129, 4096),
                                          (1000, 260), (70, 62), (2100, 128), (257, 1023), (9000, 36)])
def test_projection_backward_at_the_kernels_borders(tokens, width, fmt):
    """Both kernels of fused_rmsnorm_project_backward_q8 around the sizes where one takes over."""
    n = 4 * width
    x, W = _randn(tokens, 4, width), _randn(32, n) * 0.05
    go, proj, inv = _randn(tokens, 32), _randn(tokens, 32), torch.rand(tokens, device="cuda") + 0.5
    xc, xs = act8.quantize(x, fmt)
    gx, gW = ops.fused_rmsnorm_project_backward_q8(go, xc, xs, W, proj, inv)
    x8 = act8.dequantize(xc, xs, torch.float32).view(tokens, n).double()
    r, g, p, w = inv.double()[:, None], go.double(), proj.double(), W.double()
    s = (g * p).sum(1, keepdim=True) * r * r / n
    want = r * (g @ w) - s * x8
    # one bf16 rounding, and f32 sums of 32 products with a few more steps
    mag = r * (g.abs() @ w.abs()) + (g * p).abs().sum(1, keepdim=True) * r * r / n * x8.abs()
    assert ((gx.view(tokens, n).double() - want).abs() <= want.abs() * 2**-8 + mag * 40 * 2.0**-23 + 1e-30).all()
    gos = (go.float() * inv[:, None]).to(BF).double()
    want = gos.t() @ x8
    assert ((gW.double() - want).abs() <= want.abs() * 2**-8 + (gos.abs().t() @ x8.abs()) * ((tokens + 8) * 2.0**-23) + 1e-30).all()


# ------------------------------------------------------------- wide rows, views


@pytest.mark.parametrize("rows,width", [(3, 16376), (5, 16384), (3, 16392), (2, 16384 * 4)])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_norm_of_the_widest_rows(rows, width, dtype):
    """Against 64 bits: y and the gradients within a rounding of the type and f32 sums of `width` values."""
    x, g, w, b = _randn(rows, width, dtype=dtype), _randn(rows, width, dtype=dtype), _randn(width), _randn(width)
    y, mean, rstd = ops.layer_norm(x, w, b, 1e-5)
    X, G, W = x.double(), g.double(), w.double()
    xh = (X - X.mean(-1, keepdim=True)) * (X.var(-1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
    # A lane adds width / 1024 values or fewer, then ten levels: at most 100 roundings to 2^-24 in a
    # sum here, so statistics and sums are right to 1e-5 of their terms' magnitude (about 1 each).
    step = torch.finfo(dtype).eps / 2
    lim = lambda want, scale: step * want.abs() + 1e-5 * (1 + scale)  # noqa: E731
    Y = xh * W + b.double()
    assert ((y.double() - Y).abs() <= lim(Y, xh.abs() * W.abs())).all()
    gx, gw, gb = ops.layer_norm_backward(g, x, mean, rstd, w, b)
    gW = G * W
    GX = (gW - gW.mean(-1, keepdim=True) - xh * (gW * xh).mean(-1, keepdim=True)) * rstd.double()[:, None]
    assert ((gx.double() - GX).abs() <= lim(GX, gW.abs() + xh.abs())).all()
    for got, want, mag in ((gw, (G * xh).sum(0), (G * xh).abs().sum(0)), (gb, G.sum(0), G.abs().sum(0))):
        assert ((got.double() - want).abs() <= want.abs() * 2**-8 + 1e-5 * (1 + mag)).all()


@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,width", [(1023, 77), (1024, 1), (1024, 20), (1100, 129), (1500, 255), (1024, 257), (2000, 511),
                                        (1024, 513), (1030, 1023)])
def test_norm_of_many_rows_of_odd_width(rows, width, dtype):
    """Forward, 8-bit copy and backward from x and from codes where a warp takes a row, and beside it."""
    x, g, w, b = _randn(rows, width, dtype=dtype), _randn(rows, width, dtype=dtype), _randn(width), _randn(width)
    y, mean, rstd = ops.layer_norm(x, w, b, 1e-5)
    X, G, W = x.double(), g.double(), w.double()
    m64 = X.mean(-1, keepdim=True)
    r64 = ((X - m64).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    step = torch.finfo(dtype).eps / 2
    xh = (X - m64) * r64
    # f32 sums of at most 32 values a lane and five levels: 100 roundings to 2^-24 of their terms are 6e-6
    # of them; a row's spread may be small beside its values, which |x - mean|'s relative error follows
    err = 1e-5 * (1 + r64 * X.abs().amax(-1, keepdim=True))
    lim = lambda want, scale: step * want.abs() + err * (1 + scale)  # noqa: E731
    Y = xh * W + b.double()
    assert ((y.double() - Y).abs() <= lim(Y, xh.abs() * W.abs())).all()
    for fmt in (None, "int8", "e4m3"):
        if fmt is None:
            read, got = X, ops.layer_norm_backward(g, x, mean, rstd, w, b)
        else:
            yq, mq, rq, c, s = ops.layer_norm_q8(x, w, b, 1e-5, fmt)
            wc, wsc = act8.quantize(x, fmt)
            assert torch.equal(yq, y) and torch.equal(mq, mean) and torch.equal(rq, rstd)
            assert torch.equal(c.view(torch.uint8), wc.view(torch.uint8)) and torch.equal(s, wsc)
            read, got = act8.dequantize(c, s, torch.float32).double(), ops.layer_norm_backward_q8(g, c, s, mean, rstd, w, b)
        h = (read - mean.double()[:, None]) * rstd.double()[:, None]
        gW = G * W
        GX = (gW - gW.mean(-1, keepdim=True) - h * (gW * h).mean(-1, keepdim=True)) * rstd.double()[:, None]
        mag = rstd.double()[:, None] * (gW.abs() + gW.abs().mean(-1, keepdim=True) + h.abs() * (gW * h).abs().mean(-1, keepdim=True))
        # From codes of one column, rstd^2 = 1e5 times x's rounding passes the largest f16: a value from 65520 on
        # (half a step above 65504) rounds to infinity, so where the f32 result can lie there, infinity is right.
        inf = got[0].double() == torch.inf * GX.sign()
        over = inf & (GX.abs() + 1e-5 * mag >= 65520) & (dtype == torch.float16)
        assert (((got[0].double() - GX).abs() <= step * GX.abs() + 1e-5 * mag + 1e-7) | over).all()
        for a, want, scale in ((got[1], (G * h).sum(0), (G * h).abs().sum(0)), (got[2], G.sum(0), G.abs().sum(0))):
            assert ((a.double() - want).abs() <= want.abs() * 2**-8 + 2e-5 * scale + 1e-7).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_checkpoints_at_odd_addresses(fmt):
    """Codes and scales that are views at every odd offset give the bits of aligned ones, or, where a
    kernel for any alignment adds in another order, the same sums to f32 rounding."""
    rows, width = 40, 264
    x, g, w = _randn(rows, width), _randn(rows, width), _randn(width)
    y, mean, rstd, c, s = ops.layer_norm_q8(x, w, w, 1e-5, fmt)
    want = ops.layer_norm_backward_q8(g, c, s, mean, rstd, w, w)
    for off in (1, 2, 3, 4, 8):
        move = lambda t: torch.cat([t.view(torch.uint8).flatten().new_zeros(off), t.view(torch.uint8).flatten()])[  # noqa: E731
            off:].view(t.dtype).view(t.shape)
        for args in ((move(c), s), (c, move(s)), (move(c), move(s))):
            assert torch.equal(act8.dequantize(*args), act8.dequantize(c, s))
            got = ops.layer_norm_backward_q8(g, *args, mean, rstd, w, w)
            # bf16 results of f32 sums: one step apart at most, near zero 1e-4
            for a, b in zip(got, want):
                assert ((a.double() - b.double()).abs() <= b.double().abs() * 2**-7 + 1e-4).all()


# ------------------------------------------------------------------- graphs


def test_two_graphs_replayed_in_turn():
    """Two captured training steps of a norm (own workspaces), replayed in turn on new inputs."""
    shapes = [(300, 512), (70, 1000)]
    steps = []
    for rows, width in shapes:
        m = norm.LayerNorm(width, checkpoint_format="int8", device="cuda", dtype=BF)
        x, g = _randn(rows, width).requires_grad_(), _randn(rows, width)

        def step(m=m, x=x, g=g):
            return torch.autograd.grad(m(x), (x, m.weight, m.bias), g)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        steps.append((step, x, g, graph, out))
    for turn in range(3):
        for step, x, g, graph, out in steps:
            with torch.no_grad():
                x.copy_(_randn(*x.shape))
                g.copy_(_randn(*g.shape))
            graph.replay()
        for step, x, g, graph, out in steps:
            assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_quantising_in_a_graph():
    x = _randn(50, 4, 264)
    act8.dequantize(*act8.quantize(x, "e4m3"))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c, s = act8.quantize(x, "e4m3")
        r = act8.dequantize(c, s)
    for _ in range(2):
        x.copy_(_randn(*x.shape) * 100)
        graph.replay()
        assert torch.equal(r, act8.dequantize(*act8.quantize(x, "e4m3")))


def test_under_torch_compile():
    for fmt in (None, "int8"):
        m = norm.LayerNorm(64, device="cuda", checkpoint_format=fmt)
        f = torch.compile(lambda v: m(v * 2).sin(), backend="aot_eager", fullgraph=True)  # noqa: B023
        a, b = (_randn(4, 64, dtype=torch.float32) for _ in range(2))
        for x in (a, b):
            xe, xc = x.clone().requires_grad_(), x.clone().requires_grad_()
            ye, yc = m(xe * 2).sin(), f(xc)
            ye.sum().backward()
            yc.sum().backward()
            assert torch.equal(ye, yc) and torch.equal(xe.grad, xc.grad)
