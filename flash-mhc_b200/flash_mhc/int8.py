"""Linear layers in 8 bits for serving, and the rows of codes that they take.

A tensor's rows (its last dimension) are kept as ``codes`` (``torch.int8``) and
``scales`` (``torch.float32``, one per row): with a the row's largest magnitude,
at least 2^-100, scale = a / 127 and code = x (127 / a) rounded to nearest even.
A row with an infinity or a NaN has codes 0 and the scale NaN.  Rows of codes
start at multiples of 16 bytes: for a last dimension C that is no multiple of 16
``codes`` is a view, (..., C), of a tensor whose rows are longer.

* :func:`quantize_rows` and :func:`dequantize_rows` (ops ``row_quantize``,
  ``row_dequantize``): activations as they are, and weights (a row per output).
* :func:`rms_norm_int8` and :func:`add_rms_norm_int8` (ops of the same names):
  ``flash_mhc.norm``'s root-mean-square norm with its output in 8 bits, rounded
  once, from 32 bits to the codes.
* :func:`linear` (op ``int8_linear``): codes times a weight's codes, both scales
  and a bias.  The sums of products are exact.
* :class:`Int8Linear` and :func:`convert_linears`: the layer that a served
  ``MHCLiteBlock`` wraps, made from its trained one.

These ops have no derivative: quantising takes no part in autograd, and a backward
through the others raises.
"""

from __future__ import annotations

import copy

import torch
import torch.nn as nn
from torch._subclasses.fake_tensor import FakeTensor

from .act8 import _DTYPES, _act, _launch, _new_per_row, _register_no_derivative, _same_device, _shape
from .block import MHCLiteBlock
from .norm import RMSNorm, _params, _ptr, _residual, _weight
from .ops import _lib

ALIGN = 16  # bytes between the starts of rows of codes: a multiple of this
LEAST = 2.0 ** -100  # smallest magnitude that a scale is made for

_lib.define("row_quantize(Tensor x) -> (Tensor codes, Tensor scales)")
_lib.define("row_dequantize(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor x")
_lib.define("rms_norm_int8(Tensor x, Tensor? weight, float eps) -> (Tensor codes, Tensor scales)")
_lib.define(
    "add_rms_norm_int8(Tensor x, Tensor residual, Tensor? weight, float eps) -> (Tensor codes, Tensor scales, Tensor total)"
)
_lib.define(
    "int8_linear(Tensor codes, Tensor scales, Tensor weight_codes, Tensor weight_scales, Tensor? bias, ScalarType dtype) -> Tensor y"
)


# ------------------------------------------------------------------ arguments


def _new_codes(x: torch.Tensor) -> torch.Tensor:
    """Uninitialised codes in ``x``'s shape, rows at multiples of ALIGN bytes."""
    shape = x.shape
    pad = -shape[-1] % ALIGN
    if pad == 0:
        return torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format)
    return x.new_empty((*shape[:-1], shape[-1] + pad), dtype=torch.int8)[..., :shape[-1]]


def _new_rows(x: torch.Tensor):
    return _new_codes(x), _new_per_row(x)


def _stride(codes: torch.Tensor) -> int:
    """Bytes from row to row of a tensor that :func:`_new_codes` or :func:`_laid_out` gave."""
    shape = codes.shape
    return codes.stride(-2) if len(shape) > 1 and shape[-2] > 1 else shape[-1] + -shape[-1] % ALIGN


def _laid_out(codes: torch.Tensor) -> torch.Tensor:
    """``codes`` as (rows, C) with rows as the kernels take them: a view where they
    are so already, else a copy."""
    C = codes.shape[-1]
    t = codes if codes.dim() == 2 else codes.reshape(-1, C)
    if ((t.stride(1) == 1 or C == 1) and t.data_ptr() % ALIGN == 0
            and (t.shape[0] <= 1 or (t.stride(0) >= C and t.stride(0) % ALIGN == 0))):
        return t
    return _new_codes(t).copy_(t)


def _row_codes(op: str, name: str, codes: torch.Tensor, scales_name: str, scales: torch.Tensor):
    """(codes as (rows, C), f32 scales, row stride) of rows in 8 bits, checked."""
    if codes.dtype != torch.int8:
        raise ValueError(f"flash_mhc::{op}: {name} must be int8 (got {codes.dtype})")
    shape = codes.shape
    if not shape or shape[-1] < 1:
        raise ValueError(f"flash_mhc::{op}: {name} needs a last dimension of at least 1 (got {tuple(shape)})")
    if scales.dtype != torch.float32:
        raise ValueError(f"flash_mhc::{op}: {scales_name} must be float32 (got {scales.dtype})")
    if scales.shape != shape[:-1]:
        _shape(op, scales_name, scales, shape[:-1])
    if len(shape) == 2:  # nearly always laid out
        stride, one = codes.stride()
        if one == 1 and stride >= shape[1] and stride % ALIGN == 0 and codes.data_ptr() % ALIGN == 0:
            return codes, scales.contiguous(), stride
    codes = _laid_out(codes)
    return codes, scales.contiguous(), _stride(codes)


def _float_dtype(op: str, dtype: torch.dtype) -> int:
    if dtype not in _DTYPES:
        raise ValueError(f"flash_mhc::{op}: dtype must be float32, bfloat16 or float16 (got {dtype})")
    return _DTYPES[dtype]


# ------------------------------------------------------------------- fakes


@torch.library.register_fake("flash_mhc::row_quantize")
def _row_quantize_fake(x):
    return _new_rows(x)


@torch.library.register_fake("flash_mhc::row_dequantize")
def _row_dequantize_fake(codes, scales, dtype):
    return torch.empty(codes.shape, device=codes.device, dtype=dtype)


@torch.library.register_fake("flash_mhc::rms_norm_int8")
def _rms_norm_int8_fake(x, weight, eps):
    return _new_rows(x)


@torch.library.register_fake("flash_mhc::add_rms_norm_int8")
def _add_rms_norm_int8_fake(x, residual, weight, eps):
    return (*_new_rows(x), torch.empty(x.shape, device=x.device, dtype=x.dtype))


@torch.library.register_fake("flash_mhc::int8_linear")
def _int8_linear_fake(codes, scales, weight_codes, weight_scales, bias, dtype):
    return torch.empty((*codes.shape[:-1], weight_codes.shape[0]), device=codes.device, dtype=dtype)


# --------------------------------------------------------------------- CUDA


@torch.library.impl(_lib, "row_quantize", "CUDA")
def _row_quantize_cuda(x):
    x = _act("row_quantize", "x", x)
    codes, scales = _new_rows(x)
    _launch(x, "fmhc_row_quantize", x.data_ptr(), _DTYPES[x.dtype], codes.data_ptr(), _stride(codes),
            scales.data_ptr(), scales.numel(), x.shape[-1])
    return codes, scales


@torch.library.impl(_lib, "row_dequantize", "CUDA")
def _row_dequantize_cuda(codes, scales, dtype):
    op = "row_dequantize"
    _same_device(op, codes, scales=scales)
    out_dtype = _float_dtype(op, dtype)
    shape = codes.shape
    codes, scales, stride = _row_codes(op, "codes", codes, "scales", scales)
    x = scales.new_empty(*shape, dtype=dtype)
    _launch(codes, "fmhc_row_dequantize", codes.data_ptr(), stride, scales.data_ptr(), x.data_ptr(),
            out_dtype, codes.shape[0], codes.shape[1])
    return x


def _norm_int8(op: str, x, residual, weight, eps: float):
    x = _act(op, "x", x)
    _same_device(op, x, residual=residual, weight=weight)
    weight, pdt = _weight(op, x.shape[-1], weight)
    total = None
    if residual is not None:
        residual, total = _residual(op, x, residual), torch.empty_like(x)
    codes, scales = _new_rows(x)
    _launch(x, "fmhc_rms_norm_fwd_int8", x.data_ptr(), _DTYPES[x.dtype], _ptr(residual), _ptr(weight), pdt,
            eps, codes.data_ptr(), _stride(codes), scales.data_ptr(), _ptr(total), scales.numel(), x.shape[-1])
    return (codes, scales) if total is None else (codes, scales, total)


@torch.library.impl(_lib, "rms_norm_int8", "CUDA")
def _rms_norm_int8_cuda(x, weight, eps):
    return _norm_int8("rms_norm_int8", x, None, weight, eps)


@torch.library.impl(_lib, "add_rms_norm_int8", "CUDA")
def _add_rms_norm_int8_cuda(x, residual, weight, eps):
    return _norm_int8("add_rms_norm_int8", x, residual, weight, eps)


@torch.library.impl(_lib, "int8_linear", "CUDA")
def _int8_linear_cuda(codes, scales, weight_codes, weight_scales, bias, dtype):
    op = "int8_linear"
    _same_device(op, codes, scales=scales, weight_codes=weight_codes, weight_scales=weight_scales, bias=bias)
    y_dtype = _float_dtype(op, dtype)
    w_shape = weight_codes.shape
    if len(w_shape) != 2:
        raise ValueError(f"flash_mhc::{op}: weight_codes must be (N, K) (got {tuple(w_shape)})")
    N, K = w_shape
    lead = codes.shape[:-1]
    if codes.shape[-1:] != w_shape[1:]:
        _shape(op, "codes", codes, (*lead, K))
    codes, scales, stride = _row_codes(op, "codes", codes, "scales", scales)
    weight_codes, weight_scales, w_stride = _row_codes(op, "weight_codes", weight_codes, "weight_scales", weight_scales)
    _, bias, b_dtype = (None, None, 0) if bias is None else _params(op, N, None, bias)
    y = scales.new_empty(*lead, N, dtype=dtype)
    _launch(codes, "fmhc_int8_linear", codes.data_ptr(), stride, scales.data_ptr(), weight_codes.data_ptr(),
            w_stride, weight_scales.data_ptr(), _ptr(bias), b_dtype, y.data_ptr(), y_dtype, codes.shape[0], N, K)
    return y


# ------------------------------------------------------------------ autograd


# Outside autograd: results never require a gradient.
for _name in ("row_quantize", "row_dequantize"):
    _lib.impl(_name, torch.library.fallthrough_kernel, "Autograd")

_WHY = "it is for serving"
for _name, _impl in (
    ("rms_norm_int8", _rms_norm_int8_cuda),
    ("add_rms_norm_int8", _add_rms_norm_int8_cuda),
    ("int8_linear", _int8_linear_cuda),
):
    _register_no_derivative(_name, _impl, _WHY)


# ---------------------------------------------------------------- public names


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``x``'s rows in 8 bits: (codes, scales).  CUDA tensors of float32, bfloat16 or float16.

    Takes no part in autograd, whether or not ``x`` requires a gradient."""
    return torch.ops.flash_mhc.row_quantize(x.detach())


def dequantize_rows(codes: torch.Tensor, scales: torch.Tensor,
                    dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that (codes, scales) stand for, rounded once to ``dtype``."""
    return torch.ops.flash_mhc.row_dequantize(codes, scales.detach(), dtype)


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor | None = None,
                  eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """``norm.rms_norm``'s output as rows in 8 bits: (codes, scales)."""
    return torch.ops.flash_mhc.rms_norm_int8(x, weight, eps)


def add_rms_norm_int8(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
                      eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(codes, scales, total): ``norm.add_rms_norm`` with its norm as rows in 8 bits."""
    return torch.ops.flash_mhc.add_rms_norm_int8(x, residual, weight, eps)


def linear(codes: torch.Tensor, scales: torch.Tensor, weight_codes: torch.Tensor, weight_scales: torch.Tensor,
           bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """scales (weight_scales (codes @ weight_codes.T)) + bias in ``dtype``: a linear layer of rows in 8 bits.

    ``codes`` is (..., K) and ``weight_codes`` (N, K), K below 2^17; ``bias`` is
    float32, bfloat16 or float16.  The exact sum of products is rounded to 32 bits,
    multiplied with the weight's scale and then the row's in 32 bits, and rounded to
    ``dtype``.  Codes whose rows do not start at multiples of 16 bytes
    are copied first (those that this module makes do).
    """
    return torch.ops.flash_mhc.int8_linear(codes, scales, weight_codes, weight_scales, bias, dtype)


# -------------------------------------------------------------------- modules


def _quantize_plain(x: torch.Tensor):
    """The format on any device, in 32 bits."""
    v = x.float()
    a = v.abs().amax(-1)
    bad = ~torch.isfinite(a)
    a = a.clamp(min=LEAST)
    # Divided by tensors: torch takes 127 / a from a number by way of 1 / a, which is
    # rounded twice and sends values between two codes another way than the kernels.
    most = torch.full_like(a, 127.0)
    q = torch.where(bad.unsqueeze(-1), 0.0, v * (most / a).unsqueeze(-1)).round()
    return _new_codes(v).copy_(q), torch.where(bad, torch.nan, a / most)


def _quantize(x: torch.Tensor):
    return quantize_rows(x) if x.is_cuda and x.dtype in _DTYPES else _quantize_plain(x.detach())


class _Served(torch.autograd.Function):
    """A layer's results where a gradient of its input is wanted: a backward raises."""

    @staticmethod
    def forward(ctx, *tensors):
        ctx.set_materialize_grads(False)
        outs = tuple(t for t in tensors if not t.requires_grad)
        return outs[0].view_as(outs[0]) if len(outs) == 1 else tuple(t.view_as(t) for t in outs)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("flash_mhc: Int8Linear has no derivative (it is for serving)")


class Int8Linear(nn.Module):
    """A linear layer served in 8 bits: ``weight_codes`` (N, K), ``weight_scales`` (N,) and ``bias`` as buffers.

    ``forward(x)`` takes float activations, which are quantised row by row (the
    result has their type), or rows in 8 bits as (codes, scales) (the result has
    ``dtype``).  With a ``norm`` (an :class:`flash_mhc.norm.RMSNorm`) the layer is
    linear(norm(x)), the norm writing 8 bits at once, and ``forward(x, residual)``
    gives (linear(norm(total)), total) with total = x + residual.  On the CPU the
    same is computed with torch.  Rows of codes are laid out again when they are loaded,
    so that a state dict may hold them packed (a format that wants contiguous tensors
    takes ``weight_codes.contiguous()``).
    """

    def __init__(self, in_features: int, out_features: int, bias: bool = True, norm: RMSNorm | None = None,
                 dtype: torch.dtype = torch.bfloat16, device=None) -> None:
        super().__init__()
        if norm is not None and norm.hidden_size != in_features:
            raise ValueError(f"Int8Linear: the norm must be over {in_features} values (got {norm.hidden_size})")
        if not 0 < in_features < 1 << 17:
            raise ValueError(f"Int8Linear: in_features must be in [1, 2^17) (got {in_features})")
        _float_dtype("Int8Linear", dtype)
        self.in_features, self.out_features, self.dtype = in_features, out_features, dtype
        like = torch.empty(0, dtype=dtype, device=device)
        codes = _new_codes(like.new_empty((out_features, in_features)))
        self.register_buffer("weight_codes", codes.zero_())
        self.register_buffer("weight_scales", like.new_full((out_features,), LEAST / 127, dtype=torch.float32))
        self.register_buffer("bias", like.new_zeros((out_features,)) if bias else None)
        self.norm = norm

    @classmethod
    def from_linear(cls, layer: nn.Linear, norm: RMSNorm | None = None) -> Int8Linear:
        """The layer that stands for ``layer`` (or for ``layer`` behind ``norm``) in 8 bits."""
        w = layer.weight.detach()
        new = cls(layer.in_features, layer.out_features, layer.bias is not None, norm, w.dtype, w.device)
        new.weight_codes, new.weight_scales = _quantize(w)
        if layer.bias is not None:
            new.bias = layer.bias.detach().clone()
        new.training = layer.training  # the norm keeps its own mode
        return new

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"

    def _apply(self, fn, recurse=True):
        # A change of type is for activations and the bias: the scales stay f32.  Moving
        # the codes elsewhere packs their rows; they are laid out again.
        scales, dtype = self.weight_scales, fn(self.weight_scales.new_empty(0, dtype=self.dtype)).dtype
        super()._apply(fn, recurse)
        if self.weight_scales.dtype != torch.float32:
            self.weight_scales = scales.to(self.weight_scales.device)
        self._lay_out()
        self.dtype = dtype
        return self

    def _load_from_state_dict(self, *args, **kwargs):
        # assign=True puts the tensors of a state dict in place, whose rows may be packed.
        super()._load_from_state_dict(*args, **kwargs)
        self._lay_out()

    def _lay_out(self) -> None:
        codes = self.weight_codes
        if codes.dtype != torch.int8:
            return  # nothing that the layer takes: its forward says so
        if isinstance(codes, FakeTensor):  # has no address
            if codes.stride(0) % ALIGN:
                self.weight_codes = _new_codes(codes).copy_(codes)
            return
        self.weight_codes = _laid_out(codes)

    def _rows_of(self, x, residual):
        """(codes, scales, total or None, type of the result) of the layer's input."""
        if isinstance(x, tuple):
            if self.norm is not None or residual is not None:
                raise ValueError("Int8Linear: rows in 8 bits go to a layer without a norm, and without a residual")
            return (*x, None, self.dtype)
        if not x.is_floating_point():
            raise ValueError(f"Int8Linear: activations must be floating-point numbers (got {x.dtype})")
        norm = self.norm
        if norm is None:
            if residual is not None:
                raise ValueError("Int8Linear: a residual is added in front of the layer's norm, and it has none")
            return (*_quantize(x), None, x.dtype)
        if norm._check(x, residual):
            if residual is None:
                return (*rms_norm_int8(x, norm.weight, norm.eps), None, x.dtype)
            codes, scales, total = add_rms_norm_int8(x, residual, norm.weight, norm.eps)
            return codes, scales, total, x.dtype
        total = x if residual is None else x + residual
        v = total.float()
        y = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + norm.eps)
        if norm.weight is not None:
            y = y * norm.weight.float()
        return (*_quantize_plain(y.detach()), None if residual is None else total, x.dtype)

    def forward(self, x, residual: torch.Tensor | None = None):
        if torch.is_grad_enabled():
            wanted = [t for t in (x, residual, None if self.norm is None else self.norm.weight)
                      if isinstance(t, torch.Tensor) and t.requires_grad]
            if wanted:  # quantising leaves autograd: a backward has to say so
                with torch.no_grad():
                    out = self.forward(x, residual)
                return _Served.apply(*(out if isinstance(out, tuple) else (out,)), *wanted)
        codes, scales, total, dtype = self._rows_of(x, residual)
        if codes.is_cuda:
            # A type that the kernel has not is that of a layer that was converted as a
            # whole, or of its input: from 32 bits, as on the CPU.
            bias = self.bias
            if bias is not None and bias.dtype not in _DTYPES:
                bias = bias.float()
            y = linear(codes, scales, self.weight_codes, self.weight_scales, bias,
                       dtype if dtype in _DTYPES else torch.float32).to(dtype)
        else:
            products = codes.double() @ self.weight_codes.double().t()  # whole numbers below 2^53
            y = products.float() * self.weight_scales * scales.unsqueeze(-1)  # as the kernels order them
            y = (y if self.bias is None else y + self.bias.float()).to(dtype)
        return y if total is None else (y, total)


def convert_linears(module: nn.Module) -> nn.Module:
    """``module`` for serving, with every ``nn.Linear`` in it an :class:`Int8Linear`.

    Submodules are replaced in place; the result is ``module`` unless that is itself
    a linear layer or a ``nn.Sequential`` that gets shorter.  In a ``nn.Sequential``
    without hooks an ``RMSNorm`` in front of a linear layer becomes part of it.  The
    shorter container has the attributes, modes and names of the longer one (but is
    numbered anew if that was numbered); a layer with its norm has the layer's name.  An
    ``MHCLiteBlock`` keeps its own projection and has its wrapped layer converted.
    Subclasses of ``nn.Linear``, layers with hooks (or a ``forward`` that was set on
    them), layers of other types than float32, bfloat16 and float16 and layers of 2^17
    inputs or more stay as they are, and so do those whose weights
    ``nn.TransformerEncoderLayer`` reads itself.  A layer that stands in several places
    stays one; a norm becomes part of it if it precedes it in all of them.  An
    :class:`Int8Linear` has no ``weight``: other modules that read their linear layers'
    weights themselves cannot be converted.
    """
    return _Conversion(module).of(module)


def _has_hooks(m: nn.Module) -> bool:
    """Hooks, or a forward that was set on the module itself."""
    return "forward" in vars(m) or any(getattr(m, name) for name in (
        "_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks"))


def _shortens(m: nn.Module) -> bool:
    return type(m) is nn.Sequential and not _has_hooks(m)


class _Conversion:
    """What is known of a module's parts before and while they are replaced, by their ids.

    ``alive`` keeps the originals, so that no id becomes another's."""

    def __init__(self, root: nn.Module) -> None:
        self.alive = list(root.modules())
        self.done: dict[int, nn.Module] = {}
        self.kept: set[int] = set()  # layers whose weights their parents read
        self.before: dict[int, set[int | None]] = {id(root): {None}}  # norms in front of a layer, or none
        for m in self.alive:
            if isinstance(m, MHCLiteBlock):
                self.kept.add(id(m.W_all))
            elif isinstance(m, nn.TransformerEncoderLayer):
                self.kept.update((id(m.linear1), id(m.linear2)))
            last = None
            for child in m._modules.values():
                if child is not None:
                    self.before.setdefault(id(child), set()).add(None if last is None else id(last))
                    fits = _shortens(m) and type(child) is RMSNorm and not _has_hooks(child)
                    last = child if fits else None

    def convertible(self, m: nn.Module) -> bool:
        return (type(m) is nn.Linear and m.weight.dtype in _DTYPES and 0 < m.in_features < 1 << 17
                and not _has_hooks(m) and id(m) not in self.kept)

    def takes(self, layer: nn.Module, norm: nn.Module) -> bool:
        """Whether ``norm``, of a Sequential that may get shorter, becomes part of ``layer`` behind it."""
        return (self.before[id(layer)] == {id(norm)} and self.convertible(layer)
                and norm.hidden_size == layer.in_features)

    def of(self, module: nn.Module, norm: RMSNorm | None = None) -> nn.Module:
        """What stands in ``module``'s place (with ``norm``: in both their places)."""
        if id(module) not in self.done:
            self.done[id(module)] = module  # a module that stands in itself
            self.done[id(module)] = self._of(module, norm)
        return self.done[id(module)]

    def _of(self, module: nn.Module, norm: RMSNorm | None) -> nn.Module:
        if self.convertible(module):
            return Int8Linear.from_linear(module, norm)
        children = [(name, m) for name, m in module._modules.items() if m is not None]
        new: dict[str, nn.Module] = {}
        norm = None
        for i, (name, m) in enumerate(children):
            after = children[i + 1][1] if i + 1 < len(children) else None
            if _shortens(module) and type(m) is RMSNorm and after is not None and self.takes(after, m):
                norm = m
            else:
                new[name] = self.of(m, norm)
                norm = None
        if len(new) == len(children):
            module._modules.update(new)
            return module
        if [name for name, _ in children] == [str(i) for i in range(len(children))]:
            new = {str(i): m for i, m in enumerate(new.values())}
        shorter = nn.Sequential()
        for name, value in vars(module).items():
            if name != "_compiled_call_impl":  # runs the longer one
                shorter.__dict__[name] = copy.copy(value) if isinstance(value, (dict, set)) else value
        shorter._modules = new
        return shorter
