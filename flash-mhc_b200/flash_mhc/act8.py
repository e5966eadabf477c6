"""8-bit activation checkpoints: what a layer keeps for its backward pass, in half the bytes.

A tensor of bf16, f16 or f32 values is kept as ``codes`` (one byte per value,
``torch.int8`` or ``torch.float8_e4m3fn``) and ``scales`` (``torch.uint8``, one
byte e per block of 32 values along the last dimension, standing for
2^(e - 127)).  The scale is the smallest power of two that brings the block's
largest magnitude within the codes' range, so quantising is exact but for one
rounding of each value, and restoring is exact in bf16.  A block with an
infinity or a NaN is restored as NaN.

* :func:`quantize` and :func:`dequantize` (ops ``act_quantize``,
  ``act_dequantize``): any shape, the last dimension cut into blocks.
* ``fused_pre_map_q8``, ``fused_post_res_q8``, ``mhc_pre_forward_q8``: the
  forward mixings, which also write what their backward needs in 8 bits.
* ``pre_map_grad_h_q8``, ``post_res_grad_params_q8``,
  ``fused_rmsnorm_project_backward_q8``: their backwards, reading codes where
  the ops they are named after read bf16.

``MHCLiteBlock(..., checkpoint_format="int8")`` trains through these: its autograd
functions call them.  On their own they have no derivative (quantising has no
useful one): codes, scales and what is restored from them take no part in
autograd, and a backward through any other result raises.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from . import _native
from .ops import _bf16, _coef, _dense_like, _k2_typed_args, _lib, _n4, _on_device

BLOCK = 32  # values per scale
# format name -> (FMHC_ACT8_*, dtype of the codes)
FORMATS = {"int8": (0, torch.int8), "e4m3": (1, torch.float8_e4m3fn)}
_CODE_FORMATS = {dt: f for f, dt in FORMATS.values()}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # FMHC_DTYPE_*

_lib.define("act_quantize(Tensor x, str format) -> (Tensor codes, Tensor scales)")
_lib.define("act_dequantize(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor x")
_lib.define(
    "fused_pre_map_q8(Tensor x_streams, Tensor h_pre, str format) -> (Tensor out, Tensor x_codes, Tensor x_scales)"
)
_lib.define(
    "fused_post_res_q8(Tensor x_streams, Tensor layer_output, Tensor H_merged, Tensor h_post, str format) -> (Tensor out, Tensor lo_codes, Tensor lo_scales)"
)
_lib.define(
    "mhc_pre_forward_q8(Tensor x_streams, Tensor W, Tensor alpha_pre, Tensor alpha_post, Tensor alpha_res, Tensor bias, Tensor perm, str format) -> (Tensor layer_input, Tensor proj, Tensor inv_rms, Tensor h_pre, Tensor h_post, Tensor H_merged, Tensor x_codes, Tensor x_scales)"
)
_lib.define("pre_map_grad_h_q8(Tensor grad_out, Tensor x_codes, Tensor x_scales) -> Tensor grad_h_pre")
_lib.define(
    "post_res_grad_params_q8(Tensor grad_out, Tensor x_codes, Tensor x_scales, Tensor lo_codes, Tensor lo_scales, Tensor h_post) -> (Tensor grad_layer_output, Tensor grad_H_merged, Tensor grad_h_post)"
)
_lib.define(
    "fused_rmsnorm_project_backward_q8(Tensor grad_out, Tensor x_codes, Tensor x_scales, Tensor W, Tensor proj_out, Tensor inv_rms) -> (Tensor grad_x, Tensor grad_W)"
)


# ------------------------------------------------------------------ arguments


def _format(op: str, name: str):
    """(FMHC_ACT8_*, dtype of the codes) of a format name."""
    if name not in FORMATS:
        raise ValueError(f"flash_mhc::{op}: format must be one of {sorted(FORMATS)} (got {name!r})")
    return FORMATS[name]


def _scales_shape(shape) -> tuple:
    *rows, C = shape
    return (*rows, -(-C // BLOCK))


def _same_device(op: str, first: torch.Tensor, **others) -> None:
    """The kernels take raw pointers: every tensor has to live on ``first``'s device."""
    index = first.get_device()  # -1 on the CPU
    for name, t in others.items():
        if t is not None and t.get_device() != index:
            raise ValueError(f"flash_mhc::{op}: {name} is on {t.device}, expected {first.device}")


def _shape(op: str, name: str, t: torch.Tensor, want: tuple) -> None:
    if t.shape != want:
        raise ValueError(f"flash_mhc::{op}: {name} must be {tuple(want)} (got {tuple(t.shape)})")


def _act(op: str, name: str, x: torch.Tensor) -> torch.Tensor:
    """An activation tensor: a supported type, at least one value per row, contiguous."""
    if x.dtype not in _DTYPES:
        raise ValueError(f"flash_mhc::{op}: {name} must be float32, bfloat16 or float16 (got {x.dtype})")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"flash_mhc::{op}: {name} needs a last dimension of at least 1 (got {tuple(x.shape)})")
    return x.contiguous()


def _rows(t: torch.Tensor) -> int:
    return t.numel() // t.shape[-1]


def _checkpoint(op: str, name: str, codes: torch.Tensor, scales: torch.Tensor):
    """(codes, scales, FMHC_ACT8_*) of a checkpoint, checked against each other."""
    fmt = _CODE_FORMATS.get(codes.dtype)
    if fmt is None:
        raise ValueError(f"flash_mhc::{op}: {name} codes must be int8 or float8_e4m3fn (got {codes.dtype})")
    shape = codes.shape
    if not shape or shape[-1] < 1:
        raise ValueError(f"flash_mhc::{op}: {name} codes need a last dimension of at least 1 (got {tuple(shape)})")
    if scales.dtype != torch.uint8:
        raise ValueError(f"flash_mhc::{op}: {name} scales must be uint8 (got {scales.dtype})")
    if scales.shape != _scales_shape(shape):
        _shape(op, f"{name} scales", scales, _scales_shape(shape))
    return codes.contiguous(), scales.contiguous(), fmt


def _new_checkpoint(x: torch.Tensor, code_dtype: torch.dtype):
    if x.is_contiguous():
        return torch.empty_like(x, dtype=code_dtype), x.new_empty(_scales_shape(x.shape), dtype=torch.uint8)
    return (torch.empty_like(x, dtype=code_dtype, memory_format=torch.contiguous_format),
            x.new_empty(_scales_shape(x.shape), dtype=torch.uint8))


def _new_per_row(x: torch.Tensor) -> torch.Tensor:
    """An uninitialised f32 value per row of ``x``.  (A size that is a number is taken 1.5 us
    sooner than part of a shape.)"""
    shape = x.shape
    if len(shape) == 2:
        return x.new_empty(shape[0], dtype=torch.float32)
    return x.new_empty(shape[:-1], dtype=torch.float32)


def _launch(t: torch.Tensor, name: str, *args) -> None:
    """C-ABI call ``name`` on ``t``'s device and current stream (the last argument).

    At few tokens a call costs what Python spends on it, so the device is
    switched only if it has to be and the stream is taken as its raw handle."""
    index = t.get_device()
    if index == torch._C._cuda_getDevice():
        _native.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with _on_device(t):
            _native.call(name, *args, torch._C._cuda_getCurrentRawStream(index))


def _workspace(t: torch.Tensor, size_fn: str, *args):
    """(pointer, bytes, tensor) of the scratch that ``size_fn`` asks for on ``t``'s device."""
    n = _workspace_bytes(size_fn, t.get_device(), *args)
    ws = t.new_empty(max(n, 1), dtype=torch.uint8)
    return ws.data_ptr(), n, ws


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(size_fn: str, index: int, *args) -> int:
    """What ``size_fn`` gives for these sizes on device ``index``: always the same."""
    with torch.cuda.device(index):
        return getattr(_native.lib(), size_fn)(*args)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` at an address that is a multiple of 16 (a copy if it is a view at another one)."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _streams(op: str, name: str, x: torch.Tensor):
    if x.dim() != 3:
        raise ValueError(f"flash_mhc::{op}: {name} must be (T, n, C) (got {tuple(x.shape)})")
    _n4(op, x.shape[1])
    return x.shape


# ------------------------------------------------------------------- fakes


@torch.library.register_fake("flash_mhc::act_quantize")
def _act_quantize_fake(x, format):
    return _new_checkpoint(x, _format("act_quantize", format)[1])


@torch.library.register_fake("flash_mhc::act_dequantize")
def _act_dequantize_fake(codes, scales, dtype):
    return torch.empty(codes.shape, device=codes.device, dtype=dtype)


@torch.library.register_fake("flash_mhc::fused_pre_map_q8")
def _fused_pre_map_q8_fake(x_streams, h_pre, format):
    T, _, C = x_streams.shape
    return (x_streams.new_empty((T, C)),
            *_new_checkpoint(x_streams, _format("fused_pre_map_q8", format)[1]))


@torch.library.register_fake("flash_mhc::fused_post_res_q8")
def _fused_post_res_q8_fake(x_streams, layer_output, H_merged, h_post, format):
    return (_dense_like(x_streams),
            *_new_checkpoint(layer_output, _format("fused_post_res_q8", format)[1]))


@torch.library.register_fake("flash_mhc::mhc_pre_forward_q8")
def _mhc_pre_forward_q8_fake(x_streams, W, alpha_pre, alpha_post, alpha_res, bias, perm, format):
    T, n, C = x_streams.shape
    f = dict(device=x_streams.device, dtype=torch.float32)
    return (x_streams.new_empty((T, C)), x_streams.new_empty((T, W.shape[0])), torch.empty((T,), **f),
            torch.empty((T, 4), **f), torch.empty((T, 4), **f), torch.empty((T, 4, 4), **f),
            *_new_checkpoint(x_streams, _format("mhc_pre_forward_q8", format)[1]))


@torch.library.register_fake("flash_mhc::pre_map_grad_h_q8")
def _pre_map_grad_h_q8_fake(grad_out, x_codes, x_scales):
    T, n, C = x_codes.shape
    return torch.empty((T, n), device=x_codes.device, dtype=torch.float32)


@torch.library.register_fake("flash_mhc::post_res_grad_params_q8")
def _post_res_grad_params_q8_fake(grad_out, x_codes, x_scales, lo_codes, lo_scales, h_post):
    T, n, C = x_codes.shape
    return (grad_out.new_empty((T, C)), grad_out.new_empty((T, n, n), dtype=torch.float32),
            grad_out.new_empty((T, n), dtype=torch.float32))


@torch.library.register_fake("flash_mhc::fused_rmsnorm_project_backward_q8")
def _fused_rmsnorm_project_backward_q8_fake(grad_out, x_codes, x_scales, W, proj_out, inv_rms):
    return (torch.empty(x_codes.shape, device=x_codes.device, dtype=grad_out.dtype),
            _dense_like(W, grad_out.dtype))


# --------------------------------------------------------------------- CUDA


@torch.library.impl(_lib, "act_quantize", "CUDA")
def _act_quantize_cuda(x, format):
    fmt, code_dtype = _format("act_quantize", format)
    x = _act("act_quantize", "x", x)
    codes, scales = _new_checkpoint(x, code_dtype)
    _launch(x, "fmhc_act_quantize", x.data_ptr(), _DTYPES[x.dtype], codes.data_ptr(), fmt,
            scales.data_ptr(), _rows(x), x.shape[-1])
    return codes, scales


@torch.library.impl(_lib, "act_dequantize", "CUDA")
def _act_dequantize_cuda(codes, scales, dtype):
    op = "act_dequantize"
    _same_device(op, codes, scales=scales)
    codes, scales, fmt = _checkpoint(op, "the", codes, scales)
    if dtype not in _DTYPES:
        raise ValueError(f"flash_mhc::{op}: dtype must be float32, bfloat16 or float16 (got {dtype})")
    x = torch.empty_like(codes, dtype=dtype)
    _launch(codes, "fmhc_act_dequantize", codes.data_ptr(), fmt, scales.data_ptr(), x.data_ptr(),
            _DTYPES[dtype], _rows(codes), codes.shape[-1])
    return x


@torch.library.impl(_lib, "fused_pre_map_q8", "CUDA")
def _fused_pre_map_q8_cuda(x_streams, h_pre, format):
    op = "fused_pre_map_q8"
    fmt, code_dtype = _format(op, format)
    T, n, C = _streams(op, "x_streams", x_streams)
    _shape(op, "h_pre", h_pre, (T, n))
    _same_device(op, x_streams, h_pre=h_pre)
    x_streams, h_pre = _bf16("x_streams", x_streams), _coef(h_pre)
    out = x_streams.new_empty((T, C))
    codes, scales = _new_checkpoint(x_streams, code_dtype)
    _launch(x_streams, "fmhc_k3_fwd_q8", x_streams.data_ptr(), h_pre.data_ptr(), out.data_ptr(),
            codes.data_ptr(), scales.data_ptr(), fmt, T, n, C)
    return out, codes, scales


@torch.library.impl(_lib, "fused_post_res_q8", "CUDA")
def _fused_post_res_q8_cuda(x_streams, layer_output, H_merged, h_post, format):
    op = "fused_post_res_q8"
    fmt, code_dtype = _format(op, format)
    T, n, C = _streams(op, "x_streams", x_streams)
    _shape(op, "layer_output", layer_output, (T, C))
    _shape(op, "H_merged", H_merged, (T, n, n))
    _shape(op, "h_post", h_post, (T, n))
    _same_device(op, x_streams, layer_output=layer_output, H_merged=H_merged, h_post=h_post)
    x_streams = _bf16("x_streams", x_streams)
    layer_output = _bf16("layer_output", layer_output)
    H_merged, h_post = _coef(H_merged), _coef(h_post)
    out = torch.empty_like(x_streams)
    codes, scales = _new_checkpoint(layer_output, code_dtype)
    _launch(x_streams, "fmhc_k4_fwd_q8", x_streams.data_ptr(), layer_output.data_ptr(),
            H_merged.data_ptr(), h_post.data_ptr(), out.data_ptr(), codes.data_ptr(),
            scales.data_ptr(), fmt, T, n, C)
    return out, codes, scales


@torch.library.impl(_lib, "mhc_pre_forward_q8", "CUDA")
def _mhc_pre_forward_q8_cuda(x_streams, W, alpha_pre, alpha_post, alpha_res, bias, perm, format):
    op = "mhc_pre_forward_q8"
    fmt, code_dtype = _format(op, format)
    T, n, C = _streams(op, "x_streams", x_streams)
    _shape(op, "W", W, (32, n * C))
    _same_device(op, x_streams, W=W, alpha_pre=alpha_pre, alpha_post=alpha_post,
                 alpha_res=alpha_res, bias=bias, perm=perm)
    x_streams, W = _bf16("x_streams", x_streams), _bf16("W", W)
    args, _keep = _k2_typed_args(alpha_pre, alpha_post, alpha_res, bias, perm)
    new = lambda *shape, dtype=torch.float32: x_streams.new_empty(shape, dtype=dtype)  # noqa: E731
    layer_input, proj = new(T, C, dtype=x_streams.dtype), new(T, 32, dtype=x_streams.dtype)
    inv_rms, h_pre, h_post, H = new(T), new(T, 4), new(T, 4), new(T, 4, 4)
    codes, scales = _new_checkpoint(x_streams, code_dtype)
    # K1 and K2 in one kernel, then K3 with the checkpoint of x.
    _launch(x_streams, "fmhc_mhc_pre_fwd", x_streams.data_ptr(), W.data_ptr(), *args,
            proj.data_ptr(), inv_rms.data_ptr(), h_pre.data_ptr(), h_post.data_ptr(),
            H.data_ptr(), None, T, n, C)
    _launch(x_streams, "fmhc_k3_fwd_q8", x_streams.data_ptr(), h_pre.data_ptr(),
            layer_input.data_ptr(), codes.data_ptr(), scales.data_ptr(), fmt, T, n, C)
    return layer_input, proj, inv_rms, h_pre, h_post, H, codes, scales


@torch.library.impl(_lib, "pre_map_grad_h_q8", "CUDA")
def _pre_map_grad_h_q8_cuda(grad_out, x_codes, x_scales):
    op = "pre_map_grad_h_q8"
    T, n, C = _streams(op, "x_codes", x_codes)
    _shape(op, "grad_out", grad_out, (T, C))
    _same_device(op, grad_out, x_codes=x_codes, x_scales=x_scales)
    x_codes, x_scales, fmt = _checkpoint(op, "x", x_codes, x_scales)
    grad_out = _bf16("grad_out", grad_out)
    grad_h_pre = grad_out.new_empty((T, n), dtype=torch.float32)
    _launch(grad_out, "fmhc_k3_bwd_q8", grad_out.data_ptr(), x_codes.data_ptr(),
            x_scales.data_ptr(), fmt, grad_h_pre.data_ptr(), T, n, C)
    return grad_h_pre


@torch.library.impl(_lib, "post_res_grad_params_q8", "CUDA")
def _post_res_grad_params_q8_cuda(grad_out, x_codes, x_scales, lo_codes, lo_scales, h_post):
    op = "post_res_grad_params_q8"
    T, n, C = _streams(op, "x_codes", x_codes)
    _shape(op, "grad_out", grad_out, (T, n, C))
    _shape(op, "lo_codes", lo_codes, (T, C))
    _shape(op, "h_post", h_post, (T, n))
    _same_device(op, grad_out, x_codes=x_codes, x_scales=x_scales, lo_codes=lo_codes,
                 lo_scales=lo_scales, h_post=h_post)
    x_codes, x_scales, fmt = _checkpoint(op, "x", x_codes, x_scales)
    lo_codes, lo_scales, lo_fmt = _checkpoint(op, "lo", lo_codes, lo_scales)
    if lo_fmt != fmt:
        raise ValueError(f"flash_mhc::{op}: x_codes and lo_codes must have one format "
                         f"(got {x_codes.dtype} and {lo_codes.dtype})")
    grad_out, h_post = _bf16("grad_out", grad_out), _coef(h_post)
    grad_lo = grad_out.new_empty((T, C))
    grad_H = h_post.new_empty((T, n, n))  # h_post is f32 by now
    grad_hp = torch.empty_like(h_post)
    _launch(grad_out, "fmhc_k4_bwd_q8", grad_out.data_ptr(), x_codes.data_ptr(),
            x_scales.data_ptr(), lo_codes.data_ptr(), lo_scales.data_ptr(), fmt,
            h_post.data_ptr(), grad_lo.data_ptr(), grad_H.data_ptr(), grad_hp.data_ptr(), T, n, C)
    return grad_lo, grad_H, grad_hp


@torch.library.impl(_lib, "fused_rmsnorm_project_backward_q8", "CUDA")
def _fused_rmsnorm_project_backward_q8_cuda(grad_out, x_codes, x_scales, W, proj_out, inv_rms):
    op = "fused_rmsnorm_project_backward_q8"
    T, n, C = _streams(op, "x_codes", x_codes)
    _shape(op, "grad_out", grad_out, (T, 32))
    _shape(op, "proj_out", proj_out, (T, 32))
    _shape(op, "inv_rms", inv_rms, (T,))
    _shape(op, "W", W, (32, n * C))
    _same_device(op, grad_out, x_codes=x_codes, x_scales=x_scales, W=W, proj_out=proj_out,
                 inv_rms=inv_rms)
    x_codes, x_scales, fmt = _checkpoint(op, "x", x_codes, x_scales)
    grad_out, W, proj_out = _bf16("grad_out", grad_out), _bf16("W", W), _bf16("proj_out", proj_out)
    grad_out, W, proj_out = _aligned(grad_out), _aligned(W), _aligned(proj_out)
    x_codes, x_scales, inv_rms = _aligned(x_codes), _aligned(x_scales), _coef(inv_rms)
    grad_x, grad_W = grad_out.new_empty((T, n, C)), grad_out.new_empty((32, n * C))
    ws, ws_bytes, _keep = _workspace(grad_out, "fmhc_k1_bwd_q8_workspace_size", T, C)
    _launch(grad_out, "fmhc_k1_bwd_q8", grad_out.data_ptr(), x_codes.data_ptr(),
            x_scales.data_ptr(), fmt, W.data_ptr(), proj_out.data_ptr(), inv_rms.data_ptr(),
            grad_x.data_ptr(), grad_W.data_ptr(), ws, ws_bytes, T, n, C)
    return grad_x, grad_W


# ------------------------------------------------------------------ autograd


def _register_autograd(name: str, cuda_impl, make_function) -> None:
    """The autograd kernel of op ``name``: ``make_function(run)``'s function where a call
    records a graph (or stands inside forward-mode differentiation: the function
    refuses dual tensors), else ``run``, which takes the call on below autograd.

    It calls the CUDA implementation itself where nothing else stands between (no
    tracing, no functional or fake tensors): a second way through the dispatcher
    costs 4 us of a call's 23.  Whether that is so goes by the call's dispatch keys
    and is looked up by their bits (1.5 us less than working it out each time)."""
    op = getattr(torch.ops.flash_mhc, name).default
    below, cuda = torch._C._after_ADInplaceOrView_keyset, torch._C.DispatchKey.CUDA
    grad_enabled, any_requires_grad = torch._C.is_grad_enabled, torch._C._any_requires_grad
    direct: dict[int, bool] = {}

    def run(keyset, args):
        bits = keyset.raw_repr()
        if bits not in direct:
            direct[bits] = (keyset & below).highestPriorityTypeId() == cuda
        if direct[bits]:
            return cuda_impl(*args)
        with torch._C._AutoDispatchBelowAutograd():
            return op.redispatch(keyset & torch._C._after_autograd_keyset, *args)

    apply = make_function(run).apply

    def kernel(keyset, *args):
        if (grad_enabled() and any_requires_grad(*args)) or forward_ad._current_level >= 0:
            return apply(keyset, *args)
        if direct.get(keyset.raw_repr()):
            return cuda_impl(*args)
        return run(keyset, args)

    _lib.impl(name, kernel, "Autograd", with_keyset=True)


# Outside autograd: results never require a gradient.
for _name in ("act_quantize", "act_dequantize"):
    _lib.impl(_name, torch.library.fallthrough_kernel, "Autograd")


def _register_no_derivative(name: str, cuda_impl, why: str = "MHCLiteBlock(checkpoint_format=...) "
                            "differentiates through its own functions") -> None:
    """Op ``name``: a backward through its results raises, but for codes and scales in
    whole numbers, which are outside autograd."""

    def make_function(run):
        class NoDerivative(torch.autograd.Function):
            @staticmethod
            def forward(ctx, keyset, *args):
                out = run(keyset, args)
                outs = out if isinstance(out, tuple) else (out,)
                ctx.mark_non_differentiable(*(t for t in outs if t.dtype not in _DTYPES))
                ctx.set_materialize_grads(False)
                return out

            @staticmethod
            def backward(ctx, *_):
                raise RuntimeError(f"flash_mhc::{name} has no derivative ({why})")

        return NoDerivative

    _register_autograd(name, cuda_impl, make_function)


for _name, _impl in (
    ("fused_pre_map_q8", _fused_pre_map_q8_cuda),
    ("fused_post_res_q8", _fused_post_res_q8_cuda),
    ("mhc_pre_forward_q8", _mhc_pre_forward_q8_cuda),
    ("pre_map_grad_h_q8", _pre_map_grad_h_q8_cuda),
    ("post_res_grad_params_q8", _post_res_grad_params_q8_cuda),
    ("fused_rmsnorm_project_backward_q8", _fused_rmsnorm_project_backward_q8_cuda),
):
    _register_no_derivative(_name, _impl)


# ---------------------------------------------------------------- public names


def quantize(x: torch.Tensor, format: str = "int8") -> tuple[torch.Tensor, torch.Tensor]:
    """``x`` in 8 bits: (codes, scales).  CUDA tensors of float32, bfloat16 or float16.

    Takes no part in autograd, whether or not ``x`` requires a gradient."""
    return torch.ops.flash_mhc.act_quantize(x.detach(), format)


def dequantize(codes: torch.Tensor, scales: torch.Tensor,
               dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that (codes, scales) stand for, rounded once to ``dtype``."""
    return torch.ops.flash_mhc.act_dequantize(codes.detach(), scales, dtype)
