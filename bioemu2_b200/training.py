"""Operators for training a model next to the inference kernels: LayerNorm and the linear layer with their gradients, and
activation checkpoints in 8 bits that the backward passes take in the activation's place.

Three levels, each on the current stream of the tensors' device:

- ``layer_norm_forward`` / ``layer_norm_backward``, ``linear_forward`` / ``linear_backward``, ``checkpoint8``: the passes themselves;
- ``layer_norm`` and ``linear``: the same as differentiable functions (``checkpoint=True`` keeps ``x`` in 8 bits for backward);
- ``LayerNorm`` and ``Linear``: modules with the parameters of their ``torch.nn`` namesakes.

Scratch comes from torch's caching allocator call by call, so calls may be captured into CUDA graphs and may run at the same
time on several streams.  The order of every sum goes by the sizes alone: equal calls give equal bits.  Bad arguments raise
``ValueError`` before anything is launched.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import lib
from .functional import _ptr, _require_cuda

GROUP = 32          # neighbours in a row that share a power of two in an 8-bit checkpoint
MAX_COLS = 8192     # of a LayerNorm row
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16}


_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _code(t: torch.dtype, what: str) -> int:
    code = _DTYPES.get(t)
    if code is None:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, got {t}")
    return code


def _device(first: Tensor, *others: Tensor | None) -> int:
    """The one device of the tensors."""
    if not first.is_cuda:
        _require_cuda(first)
    device = first.get_device()
    for t in others:
        if t is not None and (not t.is_cuda or t.get_device() != device):
            _require_cuda(t)
            raise ValueError(f"tensors on {first.device} and {t.device}")
    return device


def _on_its_device(call):
    """Runs ``call`` with its tensors' device as the current one, whose current stream it launches on."""
    @functools.wraps(call)
    def run(first, *args, **kw):
        device = (first.values if isinstance(first, Checkpoint8) else first).get_device()
        if device < 0 or device == _current_device():
            return call(first, *args, **kw)
        with torch.cuda.device(device):
            return call(first, *args, **kw)
    return run


def _row_values(like: Tensor) -> Tensor:
    """One fp32 value a row of ``like``."""
    if like.ndim == 2:  # the cheapest of torch's allocating calls
        return torch.empty_strided((like.shape[0],), (1,), dtype=torch.float32, device=like.device)
    return like.new_empty(like.shape[:-1], dtype=torch.float32)


def _rows(t: Tensor, cols: int, step: int = 1) -> tuple[Tensor, int]:
    """``t`` as rows of ``cols`` neighbours and the distance of two rows in elements: the tensor's own memory where its leading
    axes lie evenly spaced (a slice of wider rows), a copy otherwise.  ``step`` > 1: rows start on 16 bytes and lie a multiple
    of ``step`` elements apart."""
    if t.is_contiguous() and (step == 1 or t.data_ptr() % 16 == 0):
        return t, cols
    try:
        rows = t.view(-1, cols)
    except RuntimeError:
        rows = None
    if rows is not None and (cols == 1 or rows.stride(1) == 1):
        pitch = rows.stride(0) if rows.shape[0] > 1 else cols
        if pitch >= cols and (step == 1 or (pitch % step == 0 and rows.data_ptr() % 16 == 0)):
            return rows, pitch
    return t.clone(memory_format=torch.contiguous_format), cols


def _parameter(t: Tensor | None, cols: int, what: str) -> Tensor | None:
    """A parameter of ``cols`` values as contiguous fp32."""
    if t is None:
        return None
    if t.shape != (cols,):
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected ({cols},)")
    if t.dtype is torch.float32 and t.is_contiguous():
        return t
    _code(t.dtype, what)
    return t.detach().float().contiguous()


class Checkpoint8(NamedTuple):
    """An activation in 8 bits: ``values`` (``float8_e4m3fn``, the activation's shape) times ``2 ** (exponents - 127)``, one
    exponent (``uint8``) for each 32 neighbours along the last axis, the last of them possibly fewer.  A group's exponent is the
    least, from -127 up, with which its largest finite magnitude is at most 448 times the power; infinities are kept as NaN.
    ``dtype`` is the activation's type."""

    values: Tensor
    exponents: Tensor
    dtype: torch.dtype

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    def restore(self, dtype: torch.dtype | None = None) -> Tensor:
        """The activation as it was kept, rounded to ``dtype`` (the activation's own)."""
        return _restore(self, dtype or self.dtype)


def _kept(kept: Checkpoint8) -> tuple[Tensor, Tensor]:
    values, exponents = kept.values, kept.exponents
    _device(values, exponents)
    if values.dtype is not torch.float8_e4m3fn or exponents.dtype is not torch.uint8:
        raise ValueError(f"a checkpoint is float8_e4m3fn with uint8 exponents, got {values.dtype} with {exponents.dtype}")
    shape = values.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"a checkpoint has rows of at least one column, got shape {tuple(shape)}")
    if exponents.shape != shape[:-1] + ((shape[-1] + GROUP - 1) // GROUP,):
        raise ValueError(f"exponents have shape {tuple(exponents.shape)}, expected one for each {GROUP} of {tuple(shape)}")
    if not values.is_contiguous() or values.data_ptr() % 16:
        values = values.clone(memory_format=torch.contiguous_format)
    return values, exponents if exponents.is_contiguous() else exponents.contiguous()


def _empty_checkpoint(x: Tensor) -> Checkpoint8:
    groups = x.shape[:-1] + ((x.shape[-1] + GROUP - 1) // GROUP,)
    return Checkpoint8(torch.empty_like(x, dtype=torch.float8_e4m3fn, memory_format=torch.contiguous_format),
                       x.new_empty(groups, dtype=torch.uint8), x.dtype)


@_on_its_device
def _restore(kept: Checkpoint8, dtype: torch.dtype) -> Tensor:
    values, exponents = _kept(kept)
    code = _code(dtype, "restored activation")
    out = torch.empty_like(values, dtype=dtype)
    if out.numel():
        cols = values.shape[-1]
        _lib.check(lib.b200_checkpoint8_restore(values.data_ptr(), exponents.data_ptr(), out.data_ptr(), values.numel() // cols, cols, code,
                                                _raw_stream(values.get_device())))
    return out


@_on_its_device
def checkpoint8(x: Tensor) -> Checkpoint8:
    """``x`` (fp32, bf16 or fp16, at least one column) in 8 bits: 1 + 1/32 bytes an element."""
    device = _device(x)
    code = _code(x.dtype, "x")
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"x has shape {tuple(x.shape)}: rows of at least one column are wanted")
    cols = x.shape[-1]
    kept = _empty_checkpoint(x)
    if x.numel():
        rows, pitch = _rows(x, cols)
        _lib.check(lib.b200_checkpoint8_fwd(rows.data_ptr(), pitch, kept.values.data_ptr(), kept.exponents.data_ptr(), x.numel() // cols,
                                            cols, code, _raw_stream(device)))
    return kept


# ---------------------------------------------------------------------------------------------------------------------------
# LayerNorm
# ---------------------------------------------------------------------------------------------------------------------------
def _norm_cols(shape, dtype: torch.dtype, other: torch.dtype) -> int:
    if len(shape) < 1 or not 1 <= shape[-1] <= MAX_COLS:
        raise ValueError(f"layer norm takes rows of 1 to {MAX_COLS} columns, got shape {tuple(shape)}")
    _code(dtype, "x")
    _code(other, "y")
    if other != dtype and dtype != torch.float32:
        raise ValueError(f"an output of another type than x wants x in float32, got {dtype} and {other}")
    return shape[-1]


@_on_its_device
def layer_norm_forward(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5,
                       out_dtype: torch.dtype | None = None, checkpoint: bool = False
                       ) -> tuple[Tensor, Tensor, Tensor, Checkpoint8 | None]:
    """``(y, mean, rstd, kept)``: ``y = (x - mean) * rstd * weight + bias`` over the last axis, fp32 statistics of shape
    ``x.shape[:-1]``, and with ``checkpoint`` ``x`` in 8 bits, written by the same pass.  An fp32 ``x`` may have ``y`` in any of the
    three types (``out_dtype``)."""
    device = _device(x, weight, bias)
    out_dtype = out_dtype or x.dtype
    cols = _norm_cols(x.shape, x.dtype, out_dtype)
    w, b = _parameter(weight, cols, "weight"), _parameter(bias, cols, "bias")
    y = torch.empty_like(x, dtype=out_dtype, memory_format=torch.contiguous_format)
    mean, rstd = _row_values(x), _row_values(x)
    kept = _empty_checkpoint(x) if checkpoint else None
    if x.numel():
        rows, pitch = _rows(x, cols)
        _lib.check(lib.b200_layer_norm_save_fwd(
            rows.data_ptr(), pitch, _ptr(w), _ptr(b), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
            kept.values.data_ptr() if kept else None, kept.exponents.data_ptr() if kept else None, x.numel() // cols, cols, eps,
            _DTYPES[x.dtype], _DTYPES[out_dtype], _raw_stream(device)))
    return y, mean, rstd, kept


@_on_its_device
def layer_norm_backward(dy: Tensor, x: Tensor | Checkpoint8, mean: Tensor, rstd: Tensor, weight: Tensor | None = None,
                        needs: tuple[bool, bool, bool] | None = None, grad_dtype: torch.dtype | None = None
                        ) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    """``(dx, dw, db)`` from the forward pass's ``mean`` and ``rstd`` and either its ``x`` or the 8-bit checkpoint of it (``dx`` then
    has the type of what was kept).  ``needs`` says which of the three are wanted: all with a weight, ``dx`` alone without one.
    ``dw`` and ``db`` have ``grad_dtype``, by default the weight's type (float32 without one)."""
    kept = x if isinstance(x, Checkpoint8) else None
    source = kept.values if kept else x
    device = _device(dy, source, mean, rstd, weight)
    shape = source.shape
    cols = _norm_cols(shape, x.dtype, dy.dtype)
    if dy.shape != shape:
        raise ValueError(f"dy has shape {tuple(dy.shape)}, x {tuple(shape)}")
    row_shape = shape[:-1]
    if mean.dtype is not torch.float32 or rstd.dtype is not torch.float32 or mean.shape != row_shape or rstd.shape != row_shape:
        raise ValueError(f"mean and rstd must be float32 of shape {tuple(row_shape)}, got {mean.dtype} {tuple(mean.shape)} and "
                         f"{rstd.dtype} {tuple(rstd.shape)}")
    if needs is None:
        needs = (True, weight is not None, weight is not None)
    grad_dtype = grad_dtype or (weight.dtype if weight is not None else torch.float32)
    grad_code = _code(grad_dtype, "the parameters' gradient")
    if not any(needs):
        return None, None, None
    w = _parameter(weight, cols, "weight")
    rows = dy.numel() // cols
    dyr, dy_pitch = _rows(dy, cols)
    values = exponents = xr = None
    x_pitch = cols
    if kept:
        values, exponents = _kept(kept)
    else:
        xr, x_pitch = _rows(x, cols)
    dx = torch.empty_like(dy, dtype=x.dtype, memory_format=torch.contiguous_format) if needs[0] else None
    dw = torch.empty_strided((cols,), (1,), dtype=grad_dtype, device=dy.device) if needs[1] else None
    db = torch.empty_strided((cols,), (1,), dtype=grad_dtype, device=dy.device) if needs[2] else None
    size = lib.b200_layer_norm_bwd_workspace_bytes(rows, cols) if needs[1] or needs[2] else 0
    scratch = torch.empty_strided((size,), (1,), dtype=torch.uint8, device=dy.device) if size else None
    _lib.check(lib.b200_layer_norm_bwd(
        dyr.data_ptr(), dy_pitch, _ptr(xr), x_pitch, _ptr(values), _ptr(exponents), mean.contiguous().data_ptr(),
        rstd.contiguous().data_ptr(), _ptr(w), _ptr(dx), _ptr(dw), _ptr(db), rows, cols, _DTYPES[x.dtype], _DTYPES[dy.dtype], grad_code,
        _ptr(scratch), size, _raw_stream(device)))
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype, checkpoint):
        y, mean, rstd, kept = layer_norm_forward(x, weight, bias, eps, out_dtype, checkpoint)
        ctx.kept_dtype = kept.dtype if kept else None
        ctx.bias_dtype = bias.dtype if bias is not None else None
        ctx.save_for_backward(kept.values if kept else x, kept.exponents if kept else None, mean, rstd, weight)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, exponents, mean, rstd, weight = ctx.saved_tensors
        if ctx.kept_dtype is not None:
            x = Checkpoint8(x, exponents, ctx.kept_dtype)
        needs = tuple(ctx.needs_input_grad[:3])
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight, needs, weight.dtype if weight is not None else ctx.bias_dtype)
        return dx, dw, db if db is None else db.to(ctx.bias_dtype), None, None, None


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5,
               out_dtype: torch.dtype | None = None, checkpoint: bool = False) -> Tensor:
    """``layer_norm_forward``'s ``y`` as a differentiable function; ``checkpoint`` keeps ``x`` in 8 bits for the backward pass."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, eps, out_dtype, checkpoint)
    return layer_norm_forward(x, weight, bias, eps, out_dtype)[0]


class LayerNorm(nn.LayerNorm):
    """``torch.nn.LayerNorm`` over the last axis with these kernels: ``out_dtype`` and ``checkpoint`` are ``layer_norm``'s."""

    def __init__(self, normalized_shape: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True,
                 out_dtype: torch.dtype | None = None, checkpoint: bool = False, device=None, dtype=None) -> None:
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1 or not 1 <= self.normalized_shape[0] <= MAX_COLS:
            raise ValueError(f"layer norm over the last axis alone, of 1 to {MAX_COLS} columns; got {self.normalized_shape}")
        self.out_dtype, self.checkpoint = out_dtype, checkpoint

    def forward(self, x: Tensor) -> Tensor:
        if x.shape[-1:] != torch.Size(self.normalized_shape):
            raise ValueError(f"x has shape {tuple(x.shape)}, its last axis must be {self.normalized_shape[0]}")
        return layer_norm(x, self.weight, self.bias, self.eps, self.out_dtype, self.checkpoint)


# ---------------------------------------------------------------------------------------------------------------------------
# Linear layer
# ---------------------------------------------------------------------------------------------------------------------------
def _linear_sizes(x_shape, x_dtype: torch.dtype, weight: Tensor, activation: str | None) -> tuple[int, int]:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(a for a in ACTIVATIONS if a)} or None, got {activation!r}")
    if x_dtype not in (torch.bfloat16, torch.float16) or weight.dtype != x_dtype:
        raise ValueError(f"x and weight must both be bfloat16 or both float16, got {x_dtype} and {weight.dtype}")
    if weight.ndim != 2 or len(x_shape) < 1 or x_shape[-1] != weight.shape[1]:
        raise ValueError(f"weight {tuple(weight.shape)} does not match x {tuple(x_shape)}")
    n, k = weight.shape
    if k % 8 or n % 8 or k < 1 or n < 1:
        raise ValueError(f"in_features={k} and out_features={n} must be positive multiples of 8")
    return k, n


@_on_its_device
def linear_forward(x: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = None,
                   residual: Tensor | None = None, out_dtype: torch.dtype | None = None, save: bool | torch.dtype = False
                   ) -> tuple[Tensor, Tensor | None]:
    """``(y, a)``: ``y = act(a) + residual`` with ``a = x @ weight.T + bias``.  ``x[..., in]`` and ``weight[out, in]`` are both bf16 or both
    fp16, ``in`` and ``out`` multiples of 8.  ``y`` has the residual's type if there is one, else ``out_dtype``: the operands' type
    (default) or fp32.  ``a`` is returned for the backward pass with ``save``: rounded to the operands' type, or with
    ``save=torch.float32`` as it is, for gradients without that rounding (None without an activation, which needs none)."""
    device = _device(x, weight, bias, residual)
    dtype = x.dtype
    k, n = _linear_sizes(x.shape, dtype, weight, activation)
    shape = x.shape[:-1] + (n,)
    if out_dtype is None:
        out_dtype = dtype if residual is None else residual.dtype
    if out_dtype is not dtype and out_dtype is not torch.float32:
        raise ValueError(f"y is {dtype} like x or float32, got {out_dtype}")
    if residual is not None and (residual.shape != shape or residual.dtype is not out_dtype):
        raise ValueError(f"residual is {residual.dtype} {tuple(residual.shape)}, y {out_dtype} {tuple(shape)}")
    save_dtype = save if isinstance(save, torch.dtype) else dtype
    if save_dtype is not dtype and save_dtype is not torch.float32:
        raise ValueError(f"the value before the activation is saved as {dtype} like x or float32, not as {save_dtype}")
    b = _parameter(bias, n, "bias")
    y = x.new_empty(shape, dtype=out_dtype)
    a = x.new_empty(shape, dtype=save_dtype) if save and activation is not None else None
    if y.numel():
        xr, x_pitch = _rows(x, k, 8)
        wr, w_pitch = _rows(weight, k, 8)
        rr, r_pitch = (None, n) if residual is None else _rows(residual, n, 8)
        _lib.check(lib.b200_linear_act_fwd(
            xr.data_ptr(), x_pitch, wr.data_ptr(), w_pitch, _ptr(b), ACTIVATIONS[activation], _ptr(rr), r_pitch, y.data_ptr(), _ptr(a),
            x.numel() // k, k, n, _DTYPES[dtype], _DTYPES[out_dtype], _DTYPES[save_dtype], _raw_stream(device)))
    return y, a


@_on_its_device
def linear_backward(dy: Tensor, x: Tensor | Checkpoint8 | None, weight: Tensor, pre: Tensor | None = None, activation: str | None = None,
                    bias: bool = True, needs: tuple[bool, bool] = (True, True), bias_dtype: torch.dtype = torch.float32
                    ) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    """``(dx, dw, db)`` of ``linear_forward`` for ``dy``, which has ``y``'s type; ``pre`` is what the forward pass saved (not needed without
    an activation), ``x`` its input or the 8-bit checkpoint of it (may be None where ``dw`` is not wanted).  ``needs`` says which of
    ``dx`` and ``dw`` are wanted, ``bias`` whether ``db`` is.  The gradient before the activation is rounded to the operands' type for the
    products, not for ``db``.  The residual's gradient is ``dy`` itself."""
    kept = x if isinstance(x, Checkpoint8) else None
    source = kept.values if kept else x
    device = _device(dy, source, weight, pre)
    if x is None and needs[1]:
        raise ValueError("the weight's gradient wants x")
    dtype, lead = (weight.dtype, dy.shape[:-1]) if x is None else (x.dtype, source.shape[:-1])
    k, n = _linear_sizes(lead + weight.shape[1:] if x is None else source.shape, dtype, weight, activation)
    shape = lead + (n,)
    if dy.shape != shape or (dy.dtype is not dtype and dy.dtype is not torch.float32):
        raise ValueError(f"dy must be {dtype} or float32 of shape {tuple(shape)}, got {dy.dtype} {tuple(dy.shape)}")
    if activation is not None and (pre is None or pre.shape != shape or (pre.dtype is not dtype and pre.dtype is not torch.float32)):
        raise ValueError(f"pre must be {dtype} or float32 of shape {tuple(shape)}, got "
                         + ("None" if pre is None else f"{pre.dtype} {tuple(pre.shape)}"))
    bias_code = _code(bias_dtype, "the bias's gradient")
    dx = weight.new_empty(lead + (k,)) if needs[0] else None
    dw = weight.new_empty((n, k)) if needs[1] else None
    db = weight.new_empty((n,), dtype=bias_dtype) if bias else None
    if dx is None and dw is None and db is None:
        return None, None, None
    g = _lib.LinearGrad()
    dyr, g.dy_pitch = _rows(dy, n, 8)
    g.dy = dyr.data_ptr()
    g.x_pitch, g.pre_pitch = k, n
    if kept:
        values, exponents = _kept(kept)
        g.values, g.exponents = values.data_ptr(), exponents.data_ptr()
    elif x is not None:
        xr, g.x_pitch = _rows(x, k, 8)
        g.x = xr.data_ptr()
    wr, g.w_pitch = _rows(weight, k, 8)
    g.w = wr.data_ptr()
    if activation is not None:
        pr, g.pre_pitch = _rows(pre, n, 8)
        g.pre, g.pre_dtype = pr.data_ptr(), _DTYPES[pre.dtype]
    g.dx, g.dw, g.db = _ptr(dx), _ptr(dw), _ptr(db)
    g.rows, g.k, g.n, g.act = dy.numel() // n, k, n, ACTIVATIONS[activation]
    g.dtype, g.dy_dtype, g.db_dtype = _DTYPES[dtype], _DTYPES[dy.dtype], bias_code
    at = ctypes.byref(g)
    size = lib.b200_linear_act_bwd_workspace_bytes(at)
    scratch = torch.empty_strided((size,), (1,), dtype=torch.uint8, device=dy.device) if size else None
    _lib.check(lib.b200_linear_act_bwd(at, _ptr(scratch), size, _raw_stream(device)))
    return dx, dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation, residual, out_dtype, checkpoint):
        y, pre = linear_forward(x, weight, bias, activation, residual, out_dtype, save=any(ctx.needs_input_grad[:3]))
        kept = checkpoint8(x) if checkpoint and ctx.needs_input_grad[1] else None
        ctx.activation, ctx.kept_dtype = activation, x.dtype if kept else None
        ctx.bias_dtype = bias.dtype if bias is not None else None
        ctx.save_for_backward(kept.values if kept else x if ctx.needs_input_grad[1] else None, kept.exponents if kept else None, weight, pre)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, exponents, weight, pre = ctx.saved_tensors
        if ctx.kept_dtype is not None:
            x = Checkpoint8(x, exponents, ctx.kept_dtype)
        dx = dw = db = None
        if any(ctx.needs_input_grad[:3]):
            dx, dw, db = linear_backward(dy, x, weight, pre, ctx.activation, ctx.needs_input_grad[2], ctx.needs_input_grad[:2],
                                         ctx.bias_dtype or torch.float32)
        return dx, dw, db, None, dy if ctx.needs_input_grad[4] else None, None, None


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = None, residual: Tensor | None = None,
           out_dtype: torch.dtype | None = None, checkpoint: bool = False) -> Tensor:
    """``linear_forward``'s ``y`` as a differentiable function; ``checkpoint`` keeps ``x`` in 8 bits for the weight's gradient."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _Linear.apply(x, weight, bias, activation, residual, out_dtype, checkpoint)
    return linear_forward(x, weight, bias, activation, residual, out_dtype)[0]


class Linear(nn.Linear):
    """``torch.nn.Linear`` with an activation and a residual in the product's epilogue, on bf16 or fp16 inputs; parameters of another
    type (fp32 masters) are rounded to the input's type at each call."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: str | None = None,
                 out_dtype: torch.dtype | None = None, checkpoint: bool = False, device=None, dtype=None) -> None:
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(a for a in ACTIVATIONS if a)} or None, got {activation!r}")
        if in_features % 8 or out_features % 8 or in_features < 1 or out_features < 1:
            raise ValueError(f"in_features={in_features} and out_features={out_features} must be positive multiples of 8")
        self.activation, self.out_dtype, self.checkpoint = activation, out_dtype, checkpoint

    def forward(self, x: Tensor, residual: Tensor | None = None) -> Tensor:
        weight = self.weight if self.weight.dtype == x.dtype else self.weight.to(x.dtype)
        return linear(x, weight, self.bias, self.activation, residual, self.out_dtype, self.checkpoint)
