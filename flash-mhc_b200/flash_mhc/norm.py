"""Norms for the layers that an mHC-lite block wraps: layer norm, with an 8-bit input checkpoint, and root-mean-square norm.

* ops ``layer_norm`` / ``layer_norm_backward``: y, mean and rstd; the gradients
  of x, weight and bias in one pass over x and the output's gradient.
* ops ``layer_norm_q8`` / ``layer_norm_backward_q8``: the same with the input
  kept in 8 bits (``flash_mhc.act8``) in x's place.  The forward's y is that of
  ``layer_norm``; only what the backward reads as x is rounded.
* :func:`layer_norm` and :class:`LayerNorm`: the differentiable function and the
  module (parameters and state_dict of ``torch.nn.LayerNorm``).

The rows are the last dimension; x is float32, bfloat16 or float16, weight and
bias (either may be missing) any of these, of one type; y has x's type, under
autocast too.  ``mean`` and ``rstd`` are not differentiable outputs, and the
gradients have no derivative of their own (asking for one raises).

From an 8-bit input the backward sees x with a rounding error, which it divides by
the row's spread: rows whose mean is much larger than their spread want x kept as
it is.  The error is, with e the scale byte and a the largest value of a block of
32, at most 2^(e - 128), which is below a / 127, for int8, and at most 2^-4 of each
value or 2^(e - 137), which is below a / 2^17, whichever is larger, for e4m3.

Root-mean-square norm (y = x / sqrt(mean(x^2) + eps) * weight):

* ops ``rms_norm`` and ``add_rms_norm``: y and rstd; with a residual, of
  total = x + residual rounded to x's type, which is returned too.
* op ``rms_norm_backward``: the gradients of what is normalised, to which the
  gradient of total is added, and of weight, in one pass.
* :func:`rms_norm`, :func:`add_rms_norm` and :class:`RMSNorm` (parameters and
  state_dict of ``torch.nn.RMSNorm``).  Types, ``rstd`` and second derivatives
  are as for layer norm; its output in 8 bits is in ``flash_mhc.int8``.
"""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from .act8 import (_DTYPES, _act, _checkpoint, _format, _launch, _new_checkpoint, _new_per_row, _register_autograd,
                   _rows, _same_device, _shape, _workspace)
from .ops import _lib

_lib.define(
    "layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor y, Tensor mean, Tensor rstd)"
)
_lib.define(
    "layer_norm_q8(Tensor x, Tensor? weight, Tensor? bias, float eps, str format) -> (Tensor y, Tensor mean, Tensor rstd, Tensor codes, Tensor scales)"
)
# grad_weight and grad_bias are empty where the parameter is missing.
_lib.define(
    "layer_norm_backward(Tensor grad_out, Tensor x, Tensor mean, Tensor rstd, Tensor? weight, Tensor? bias) -> (Tensor grad_x, Tensor grad_weight, Tensor grad_bias)"
)
_lib.define(
    "layer_norm_backward_q8(Tensor grad_out, Tensor codes, Tensor scales, Tensor mean, Tensor rstd, Tensor? weight, Tensor? bias) -> (Tensor grad_x, Tensor grad_weight, Tensor grad_bias)"
)
_lib.define("rms_norm(Tensor x, Tensor? weight, float eps) -> (Tensor y, Tensor rstd)")
_lib.define(
    "add_rms_norm(Tensor x, Tensor residual, Tensor? weight, float eps) -> (Tensor y, Tensor total, Tensor rstd)"
)
# x: what was normalised (add_rms_norm's total).  grad_weight is empty where the weight is missing.
_lib.define(
    "rms_norm_backward(Tensor grad_out, Tensor? grad_total, Tensor x, Tensor rstd, Tensor? weight) -> (Tensor grad_x, Tensor grad_weight)"
)


def _params(op: str, C: int, weight, bias):
    """weight and bias as contiguous (C,) tensors of one type, and that type's FMHC_DTYPE_*."""
    dt = 0
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            _shape(op, name, p, (C,))
            if p.dtype not in _DTYPES:
                raise ValueError(f"flash_mhc::{op}: {name} must be float32, bfloat16 or float16 (got {p.dtype})")
            dt = _DTYPES[p.dtype]
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"flash_mhc::{op}: weight and bias must have one type (got {weight.dtype} and {bias.dtype})")
    return (None if weight is None else weight.contiguous(), None if bias is None else bias.contiguous(), dt)


def _weight(op: str, C: int, weight):
    """``weight`` as _params gives it, by a shorter way where nothing is wrong with it."""
    if weight is None:
        return None, 0
    if len(weight.shape) == 1 and weight.shape[0] == C and weight.dtype in _DTYPES:
        return weight.contiguous(), _DTYPES[weight.dtype]
    weight, _, dt = _params(op, C, weight, None)
    return weight, dt


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stats(op: str, mean, rstd, rows_shape):
    for name, t in (("mean", mean), ("rstd", rstd)):
        _shape(op, name, t, rows_shape)
        if t.dtype != torch.float32:
            raise ValueError(f"flash_mhc::{op}: {name} must be float32 (got {t.dtype})")
    return mean.contiguous(), rstd.contiguous()


def _forward(op: str, x, weight, bias, eps: float, format=None):
    x = _act(op, "x", x)
    _same_device(op, x, weight=weight, bias=bias)
    weight, bias, pdt = _params(op, x.shape[-1], weight, bias)
    y = torch.empty_like(x)
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    fmt, codes, scales = -1, None, None
    if format is not None:
        fmt, code_dtype = _format(op, format)
        codes, scales = _new_checkpoint(x, code_dtype)
    _launch(x, "fmhc_layer_norm_fwd", x.data_ptr(), _DTYPES[x.dtype], _ptr(weight), _ptr(bias), pdt,
            eps, y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), _ptr(codes), fmt, _ptr(scales),
            _rows(x), x.shape[-1])
    return (y, mean, rstd) if format is None else (y, mean, rstd, codes, scales)


def _backward(op: str, grad_out, x, codes, scales, mean, rstd, weight, bias):
    grad_out = _act(op, "grad_out", grad_out)
    _same_device(op, grad_out, x=x, codes=codes, scales=scales, mean=mean, rstd=rstd, weight=weight,
                 bias=bias)
    fmt = -1
    if codes is None:
        _shape(op, "x", x, grad_out.shape)
        if x.dtype != grad_out.dtype:
            raise ValueError(f"flash_mhc::{op}: grad_out and x must have one type (got {grad_out.dtype} and {x.dtype})")
        x = x.contiguous()
    else:
        _shape(op, "codes", codes, grad_out.shape)
        codes, scales, fmt = _checkpoint(op, "the", codes, scales)
    mean, rstd = _stats(op, mean, rstd, grad_out.shape[:-1])
    C, rows = grad_out.shape[-1], _rows(grad_out)
    weight, bias, pdt = _params(op, C, weight, bias)
    grad_x = torch.empty_like(grad_out)
    none = lambda: grad_out.new_empty((0,), dtype=torch.float32)  # noqa: E731
    grad_w = none() if weight is None else torch.empty_like(weight)
    grad_b = none() if bias is None else torch.empty_like(bias)
    ws, ws_bytes, _keep = None, 0, None
    if weight is not None or bias is not None:
        ws, ws_bytes, _keep = _workspace(grad_out, "fmhc_layer_norm_bwd_workspace_size", rows, C)
    _launch(grad_out, "fmhc_layer_norm_bwd", grad_out.data_ptr(), _DTYPES[grad_out.dtype], _ptr(x),
            _ptr(codes), fmt, _ptr(scales), mean.data_ptr(), rstd.data_ptr(), _ptr(weight), pdt,
            grad_x.data_ptr(), None if weight is None else grad_w.data_ptr(),
            None if bias is None else grad_b.data_ptr(), ws, ws_bytes, rows, C)
    return grad_x, grad_w, grad_b


def _residual(op: str, x, residual):
    """``residual`` beside ``x`` (already checked): of its shape and type, contiguous."""
    if residual.shape != x.shape:
        _shape(op, "residual", residual, x.shape)
    if residual.dtype != x.dtype:
        raise ValueError(f"flash_mhc::{op}: x and residual must have one type (got {x.dtype} and {residual.dtype})")
    return residual.contiguous()


def _rms_forward(op: str, x, residual, weight, eps: float):
    x = _act(op, "x", x)
    _same_device(op, x, residual=residual, weight=weight)
    C = x.shape[-1]
    weight, pdt = _weight(op, C, weight)
    total = None
    if residual is not None:
        residual, total = _residual(op, x, residual), torch.empty_like(x)
    y, rstd = torch.empty_like(x), _new_per_row(x)
    _launch(x, "fmhc_rms_norm_fwd", x.data_ptr(), _DTYPES[x.dtype], _ptr(residual), _ptr(weight), pdt,
            eps, y.data_ptr(), _ptr(total), rstd.data_ptr(), x.numel() // C, C)
    return (y, rstd) if total is None else (y, total, rstd)


def _rms_backward(op: str, grad_out, grad_total, x, rstd, weight):
    grad_out = _act(op, "grad_out", grad_out)
    _same_device(op, grad_out, grad_total=grad_total, x=x, rstd=rstd, weight=weight)
    shape, dtype = grad_out.shape, grad_out.dtype
    for name, t in (("x", x), ("grad_total", grad_total)):
        if t is not None and (t.shape != shape or t.dtype != dtype):
            _shape(op, name, t, shape)
            raise ValueError(f"flash_mhc::{op}: grad_out and {name} must have one type (got {dtype} and {t.dtype})")
    x = x.contiguous()
    grad_total = None if grad_total is None else grad_total.contiguous()
    if rstd.shape != shape[:-1]:
        _shape(op, "rstd", rstd, shape[:-1])
    if rstd.dtype != torch.float32:
        raise ValueError(f"flash_mhc::{op}: rstd must be float32 (got {rstd.dtype})")
    rstd = rstd.contiguous()
    C, rows = shape[-1], grad_out.numel() // shape[-1]
    weight, pdt = _weight(op, C, weight)
    grad_x = torch.empty_like(grad_out)
    ws, ws_bytes, _keep = None, 0, None
    if weight is None:
        grad_w = grad_out.new_empty((0,), dtype=torch.float32)
    else:
        grad_w = torch.empty_like(weight)
        ws, ws_bytes, _keep = _workspace(grad_out, "fmhc_rms_norm_bwd_workspace_size", rows, C)
    _launch(grad_out, "fmhc_rms_norm_bwd", grad_out.data_ptr(), _DTYPES[dtype], _ptr(grad_total),
            x.data_ptr(), rstd.data_ptr(), _ptr(weight), pdt, grad_x.data_ptr(),
            None if weight is None else grad_w.data_ptr(), ws, ws_bytes, rows, C)
    return grad_x, grad_w


# -------------------------------------------------------------------- fakes


@torch.library.register_fake("flash_mhc::layer_norm")
def _layer_norm_fake(x, weight, bias, eps):
    stats = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    return torch.empty(x.shape, device=x.device, dtype=x.dtype), stats, torch.empty_like(stats)


@torch.library.register_fake("flash_mhc::layer_norm_q8")
def _layer_norm_q8_fake(x, weight, bias, eps, format):
    return (*_layer_norm_fake(x, weight, bias, eps),
            *_new_checkpoint(x, _format("layer_norm_q8", format)[1]))


@torch.library.register_fake("flash_mhc::layer_norm_backward")
def _layer_norm_backward_fake(grad_out, x, mean, rstd, weight, bias):
    none = lambda: torch.empty(0, device=grad_out.device, dtype=torch.float32)  # noqa: E731
    return (torch.empty(grad_out.shape, device=grad_out.device, dtype=grad_out.dtype),
            none() if weight is None else torch.empty_like(weight),
            none() if bias is None else torch.empty_like(bias))


@torch.library.register_fake("flash_mhc::layer_norm_backward_q8")
def _layer_norm_backward_q8_fake(grad_out, codes, scales, mean, rstd, weight, bias):
    return _layer_norm_backward_fake(grad_out, codes, mean, rstd, weight, bias)


@torch.library.register_fake("flash_mhc::rms_norm")
def _rms_norm_fake(x, weight, eps):
    return (torch.empty(x.shape, device=x.device, dtype=x.dtype),
            torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32))


@torch.library.register_fake("flash_mhc::add_rms_norm")
def _add_rms_norm_fake(x, residual, weight, eps):
    y, rstd = _rms_norm_fake(x, weight, eps)
    return y, torch.empty_like(y), rstd


@torch.library.register_fake("flash_mhc::rms_norm_backward")
def _rms_norm_backward_fake(grad_out, grad_total, x, rstd, weight):
    return (torch.empty(grad_out.shape, device=grad_out.device, dtype=grad_out.dtype),
            torch.empty(0, device=grad_out.device, dtype=torch.float32) if weight is None
            else torch.empty(weight.shape, device=weight.device, dtype=weight.dtype))


# --------------------------------------------------------------------- CUDA


@torch.library.impl(_lib, "layer_norm", "CUDA")
def _layer_norm_cuda(x, weight, bias, eps):
    return _forward("layer_norm", x, weight, bias, eps)


@torch.library.impl(_lib, "layer_norm_q8", "CUDA")
def _layer_norm_q8_cuda(x, weight, bias, eps, format):
    return _forward("layer_norm_q8", x, weight, bias, eps, format)


@torch.library.impl(_lib, "layer_norm_backward", "CUDA")
def _layer_norm_backward_cuda(grad_out, x, mean, rstd, weight, bias):
    return _backward("layer_norm_backward", grad_out, x, None, None, mean, rstd, weight, bias)


@torch.library.impl(_lib, "layer_norm_backward_q8", "CUDA")
def _layer_norm_backward_q8_cuda(grad_out, codes, scales, mean, rstd, weight, bias):
    return _backward("layer_norm_backward_q8", grad_out, None, codes, scales, mean, rstd, weight, bias)


@torch.library.impl(_lib, "rms_norm", "CUDA")
def _rms_norm_cuda(x, weight, eps):
    return _rms_forward("rms_norm", x, None, weight, eps)


@torch.library.impl(_lib, "add_rms_norm", "CUDA")
def _add_rms_norm_cuda(x, residual, weight, eps):
    return _rms_forward("add_rms_norm", x, residual, weight, eps)


@torch.library.impl(_lib, "rms_norm_backward", "CUDA")
def _rms_norm_backward_cuda(grad_out, grad_total, x, rstd, weight):
    return _rms_backward("rms_norm_backward", grad_out, grad_total, x, rstd, weight)


# ------------------------------------------------------------------ autograd


class _GradsOnce(torch.autograd.Function):
    """The gradients where a graph of them is asked for: they have no derivative here, and say so.

    ``mark`` requires a gradient, so that the result does, whatever the arguments do
    (codes never do, although they depend on x)."""

    @staticmethod
    def forward(ctx, mark, name, op, *args):
        ctx.name = name
        return op(*args)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"flash_mhc::{ctx.name} has no second derivative")


def _grads(name: str, op, gy, *args):
    """The gradients that ``op`` gives, by way of _GradsOnce under create_graph=True."""
    if torch.is_grad_enabled():
        return _GradsOnce.apply(gy.new_empty(0).requires_grad_(), name, op, gy, *args)
    return op(gy, *args)


def _register_norm(name: str, cuda_impl, backward: str, kept) -> None:
    """Op ``name``: ``kept`` picks what the backward reads in x's place."""
    backward_op = getattr(torch.ops.flash_mhc, backward)

    def make_function(run):
        class LayerNormFunction(torch.autograd.Function):
            @staticmethod
            def forward(ctx, keyset, *args):
                out = run(keyset, args)
                ctx.save_for_backward(*kept(args[0], out), out[1], out[2], args[1], args[2])
                ctx.mark_non_differentiable(*out[1:])
                ctx.set_materialize_grads(False)  # no zeros in the size of the codes
                ctx.rest = (None,) * (len(args) - 3)
                return out

            @staticmethod
            def backward(ctx, gy, *_):
                if gy is None:
                    return (None, None, None, None, *ctx.rest)
                grads = _grads("layer_norm", backward_op, gy, *ctx.saved_tensors)
                need = ctx.needs_input_grad[1:]
                return (None, *(g if n else None for g, n in zip(grads, need)), *ctx.rest)

        return LayerNormFunction

    _register_autograd(name, cuda_impl, make_function)


_register_norm("layer_norm", _layer_norm_cuda, "layer_norm_backward", lambda x, out: (x,))
_register_norm("layer_norm_q8", _layer_norm_q8_cuda, "layer_norm_backward_q8", lambda x, out: out[3:])


def _register_rms_norm(name: str, cuda_impl, add: bool) -> None:
    """Op ``name``: keeps what it normalised, which is x, or with ``add`` its output total."""
    backward_op = torch.ops.flash_mhc.rms_norm_backward

    def make_function(run):
        class RMSNormFunction(torch.autograd.Function):
            @staticmethod
            def forward(ctx, keyset, *args):
                out = run(keyset, args)
                ctx.save_for_backward(out[1] if add else args[0], out[-1], args[-2])
                ctx.mark_non_differentiable(out[-1])
                ctx.set_materialize_grads(False)
                return out

            @staticmethod
            def backward(ctx, gy, *rest):
                gt = rest[0] if add else None
                if gy is None:  # nothing through the norm
                    gx, gw = gt, None
                else:
                    x, rstd, weight = ctx.saved_tensors
                    gx, gw = _grads(name, backward_op, gy, gt, x, rstd, weight)
                need = ctx.needs_input_grad[1:]
                grads = (gx, gx, gw) if add else (gx, gw)
                return (None, *(g if n else None for g, n in zip(grads, need)), None)

        return RMSNormFunction

    _register_autograd(name, cuda_impl, make_function)


_register_rms_norm("rms_norm", _rms_norm_cuda, add=False)
_register_rms_norm("add_rms_norm", _add_rms_norm_cuda, add=True)


# ---------------------------------------------------------------- public names


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5, checkpoint_format: str | None = None) -> torch.Tensor:
    """Layer norm over the last dimension of a CUDA tensor, differentiable in x, weight and bias.

    With ``checkpoint_format`` ("int8" or "e4m3") a call that records a graph
    keeps x in 8 bits for the backward pass instead of x itself.
    """
    if checkpoint_format is not None:
        _format("layer_norm", checkpoint_format)
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
            return torch.ops.flash_mhc.layer_norm_q8(x, weight, bias, eps, checkpoint_format)[0]
    return torch.ops.flash_mhc.layer_norm(x, weight, bias, eps)[0]


class LayerNorm(nn.Module):
    """``torch.nn.LayerNorm`` over the last dimension, with the same parameters and state_dict.

    CUDA inputs of float32, bfloat16 or float16 take the fused kernels (and keep
    their input in ``checkpoint_format``, if given); every other input takes
    ``torch.nn.functional.layer_norm``, which keeps it as it is.
    """

    def __init__(self, hidden_size: int, eps: float = 1e-5, elementwise_affine: bool = True,
                 bias: bool = True, checkpoint_format: str | None = None, device=None,
                 dtype=None) -> None:
        super().__init__()
        if checkpoint_format is not None:
            _format("layer_norm", checkpoint_format)
        self.hidden_size = hidden_size
        self.eps = eps
        self.checkpoint_format = checkpoint_format
        f = dict(device=device, dtype=dtype)
        affine = elementwise_affine
        self.weight = nn.Parameter(torch.ones(hidden_size, **f)) if affine else None
        self.bias = nn.Parameter(torch.zeros(hidden_size, **f)) if affine and bias else None

    def extra_repr(self) -> str:
        return f"{self.hidden_size}, eps={self.eps}, checkpoint_format={self.checkpoint_format}"

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1:] != (self.hidden_size,):
            raise ValueError(f"LayerNorm: expected a last dimension of {self.hidden_size} (got {tuple(x.shape)})")
        if x.is_cuda and x.dtype in _DTYPES:
            return layer_norm(x, self.weight, self.bias, self.eps, self.checkpoint_format)
        return F.layer_norm(x, (self.hidden_size,), self.weight, self.bias, self.eps)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """Root-mean-square norm over the last dimension of a CUDA tensor, differentiable in x and weight."""
    return torch.ops.flash_mhc.rms_norm(x, weight, eps)[0]


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
                 eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """(rms_norm(total), total) with total = x + residual rounded to x's type, in one pass.

    Differentiable in x, residual and weight; x and residual have one shape and type.
    """
    return torch.ops.flash_mhc.add_rms_norm(x, residual, weight, eps)[:2]


class RMSNorm(nn.Module):
    """``torch.nn.RMSNorm`` over the last dimension, with the same parameter and state_dict.

    ``forward(x)`` gives y, ``forward(x, residual)`` (y, total) with
    total = x + residual.  CUDA inputs of float32, bfloat16 or float16 take the
    fused kernels, every other input torch's.
    """

    def __init__(self, hidden_size: int, eps: float = 1e-6, elementwise_affine: bool = True, device=None,
                 dtype=None) -> None:
        super().__init__()
        self.hidden_size = hidden_size
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype)) if elementwise_affine else None

    def extra_repr(self) -> str:
        return f"{self.hidden_size}, eps={self.eps}"

    def _check(self, x: torch.Tensor, residual: torch.Tensor | None) -> bool:
        """Whether the fused kernels take ``x``."""
        if x.shape[-1:] != (self.hidden_size,):
            raise ValueError(f"RMSNorm: expected a last dimension of {self.hidden_size} (got {tuple(x.shape)})")
        if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
            raise ValueError(f"RMSNorm: the residual must be {tuple(x.shape)} and {x.dtype} like x "
                             f"(got {tuple(residual.shape)} and {residual.dtype})")
        return x.is_cuda and x.dtype in _DTYPES

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        if self._check(x, residual):
            if residual is None:
                return rms_norm(x, self.weight, self.eps)
            return add_rms_norm(x, residual, self.weight, self.eps)
        total = x if residual is None else x + residual
        y = F.rms_norm(total, (self.hidden_size,), self.weight, self.eps)
        return y if residual is None else (y, total)
