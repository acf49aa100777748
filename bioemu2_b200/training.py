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

import contextlib
import ctypes
from typing import NamedTuple

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import lib
from .functional import _ptr, _require_cuda, _stream

GROUP = 32          # neighbours in a row that share a power of two in an 8-bit checkpoint
MAX_COLS = 8192     # of a LayerNorm row
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16}


def _on(device: torch.device):
    """The tensors' device as the current one (and so its current stream as the one that is launched on)."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _code(t: torch.dtype, what: str) -> int:
    code = _DTYPES.get(t)
    if code is None:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, got {t}")
    return code


def _same_device(first: Tensor, *others: Tensor | None) -> None:
    _require_cuda(first)
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f"tensors on {first.device} and {t.device}")


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
    if tuple(t.shape) != (cols,):
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected ({cols},)")
    _code(t.dtype, what)
    t = t.detach()
    return t.contiguous() if t.dtype == torch.float32 else t.float().contiguous()


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
        values, exponents = _kept(self)
        out = torch.empty(values.shape, dtype=dtype or self.dtype, device=values.device)
        code = _code(out.dtype, "restored activation")
        if out.numel():
            cols = values.shape[-1]
            with _on(values.device):
                _lib.check(lib.b200_checkpoint8_restore(values.data_ptr(), exponents.data_ptr(), out.data_ptr(), values.numel() // cols,
                                                        cols, code, _stream()))
        return out


def _kept(kept: Checkpoint8) -> tuple[Tensor, Tensor]:
    values, exponents = kept.values, kept.exponents
    _same_device(values, exponents)
    if values.dtype != torch.float8_e4m3fn or exponents.dtype != torch.uint8:
        raise ValueError(f"a checkpoint is float8_e4m3fn with uint8 exponents, got {values.dtype} with {exponents.dtype}")
    if values.ndim < 1 or values.shape[-1] < 1:
        raise ValueError(f"a checkpoint has rows of at least one column, got shape {tuple(values.shape)}")
    want = values.shape[:-1] + ((values.shape[-1] + GROUP - 1) // GROUP,)
    if exponents.shape != want:
        raise ValueError(f"exponents have shape {tuple(exponents.shape)}, expected {tuple(want)}")
    values = values.contiguous()
    return (values if values.data_ptr() % 16 == 0 else values.clone()), exponents.contiguous()


def _empty_checkpoint(x: Tensor) -> Checkpoint8:
    values = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    exponents = torch.empty(x.shape[:-1] + ((x.shape[-1] + GROUP - 1) // GROUP,), dtype=torch.uint8, device=x.device)
    return Checkpoint8(values, exponents, x.dtype)


def checkpoint8(x: Tensor) -> Checkpoint8:
    """``x`` (fp32, bf16 or fp16, at least one column) in 8 bits: 1 + 1/32 bytes an element."""
    _require_cuda(x)
    code = _code(x.dtype, "x")
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"x has shape {tuple(x.shape)}: rows of at least one column are wanted")
    x = x.detach()
    cols = x.shape[-1]
    kept = _empty_checkpoint(x)
    if x.numel():
        with _on(x.device):
            rows, pitch = _rows(x, cols)
            _lib.check(lib.b200_checkpoint8_fwd(rows.data_ptr(), pitch, kept.values.data_ptr(), kept.exponents.data_ptr(),
                                                x.numel() // cols, cols, code, _stream()))
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


def layer_norm_forward(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5,
                       out_dtype: torch.dtype | None = None, checkpoint: bool = False
                       ) -> tuple[Tensor, Tensor, Tensor, Checkpoint8 | None]:
    """``(y, mean, rstd, kept)``: ``y = (x - mean) * rstd * weight + bias`` over the last axis, fp32 statistics of shape
    ``x.shape[:-1]``, and with ``checkpoint`` ``x`` in 8 bits, written by the same pass.  An fp32 ``x`` may have ``y`` in any of the
    three types (``out_dtype``)."""
    _same_device(x, weight, bias)
    x = x.detach()
    out_dtype = out_dtype or x.dtype
    cols = _norm_cols(x.shape, x.dtype, out_dtype)
    with _on(x.device):
        w, b = _parameter(weight, cols, "weight"), _parameter(bias, cols, "bias")
        y = torch.empty(x.shape, dtype=out_dtype, device=x.device)
        mean, rstd = torch.empty((2,) + x.shape[:-1], dtype=torch.float32, device=x.device).unbind(0)
        kept = _empty_checkpoint(x) if checkpoint else None
        if x.numel():
            rows, pitch = _rows(x, cols)
            _lib.check(lib.b200_layer_norm_save_fwd(
                rows.data_ptr(), pitch, _ptr(w), _ptr(b), y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                kept.values.data_ptr() if kept else None, kept.exponents.data_ptr() if kept else None, x.numel() // cols, cols, eps,
                _DTYPES[x.dtype], _DTYPES[out_dtype], _stream()))
    return y, mean, rstd, kept


def layer_norm_backward(dy: Tensor, x: Tensor | Checkpoint8, mean: Tensor, rstd: Tensor, weight: Tensor | None = None,
                        needs: tuple[bool, bool, bool] | None = None, grad_dtype: torch.dtype | None = None
                        ) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    """``(dx, dw, db)`` from the forward pass's ``mean`` and ``rstd`` and either its ``x`` or the 8-bit checkpoint of it (``dx`` then
    has the type of what was kept).  ``needs`` says which of the three are wanted: all with a weight, ``dx`` alone without one.
    ``dw`` and ``db`` have ``grad_dtype``, by default the weight's type (float32 without one)."""
    kept = x if isinstance(x, Checkpoint8) else None
    source = kept.values if kept else x
    _same_device(dy, source, mean, rstd, weight)
    cols = _norm_cols(source.shape, x.dtype, dy.dtype)
    if dy.shape != source.shape:
        raise ValueError(f"dy has shape {tuple(dy.shape)}, x {tuple(source.shape)}")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or t.shape != source.shape[:-1]:
            raise ValueError(f"{name} must be float32 of shape {tuple(source.shape[:-1])}, got {t.dtype} {tuple(t.shape)}")
    needs = needs or (True, weight is not None, weight is not None)
    grad_dtype = grad_dtype or (weight.dtype if weight is not None else torch.float32)
    grad_code = _code(grad_dtype, "the parameters' gradient")
    with _on(dy.device):
        dy = dy.detach()
        w = _parameter(weight, cols, "weight")
        new = dict(device=dy.device)
        dx = torch.empty(dy.shape, dtype=x.dtype, **new) if needs[0] else None
        dw = torch.empty(cols, dtype=grad_dtype, **new) if needs[1] else None
        db = torch.empty(cols, dtype=grad_dtype, **new) if needs[2] else None
        if not any(needs):
            return None, None, None
        rows = dy.numel() // cols
        dyr, dy_pitch = _rows(dy, cols)
        values = exponents = xr = None
        x_pitch = cols
        if kept:
            values, exponents = _kept(kept)
        else:
            xr, x_pitch = _rows(x.detach(), cols)
        mean, rstd = mean.contiguous(), rstd.contiguous()
        size = lib.b200_layer_norm_bwd_workspace_bytes(rows, cols) if needs[1] or needs[2] else 0
        scratch = torch.empty(size, dtype=torch.uint8, **new) if size else None
        _lib.check(lib.b200_layer_norm_bwd(
            _ptr(dyr), dy_pitch, _ptr(xr), x_pitch, _ptr(values), _ptr(exponents), mean.data_ptr(), rstd.data_ptr(), _ptr(w), _ptr(dx),
            _ptr(dw), _ptr(db), rows, cols, _DTYPES[x.dtype], _DTYPES[dy.dtype], grad_code, _ptr(scratch), size, _stream()))
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


def linear_forward(x: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = None,
                   residual: Tensor | None = None, out_dtype: torch.dtype | None = None, save: bool = False
                   ) -> tuple[Tensor, Tensor | None]:
    """``(y, a)``: ``y = act(a) + residual`` with ``a = x @ weight.T + bias``.  ``x[..., in]`` and ``weight[out, in]`` are both bf16 or both
    fp16, ``in`` and ``out`` multiples of 8.  ``y`` has the residual's type if there is one, else ``out_dtype``: the operands' type
    (default) or fp32.  ``a``, rounded to the operands' type, is returned for the backward pass with ``save`` (None without an
    activation, which needs none)."""
    _same_device(x, weight, bias, residual)
    k, n = _linear_sizes(x.shape, x.dtype, weight, activation)
    shape = x.shape[:-1] + (n,)
    out_dtype = out_dtype or (residual.dtype if residual is not None else x.dtype)
    if out_dtype not in (x.dtype, torch.float32):
        raise ValueError(f"y is {x.dtype} like x or float32, got {out_dtype}")
    if residual is not None and (residual.shape != shape or residual.dtype != out_dtype):
        raise ValueError(f"residual is {residual.dtype} {tuple(residual.shape)}, y {out_dtype} {tuple(shape)}")
    with _on(x.device):
        b = _parameter(bias, n, "bias")
        y = torch.empty(shape, dtype=out_dtype, device=x.device)
        a = torch.empty(shape, dtype=x.dtype, device=x.device) if save and activation is not None else None
        if y.numel():
            xr, x_pitch = _rows(x.detach(), k, 8)
            wr, w_pitch = _rows(weight.detach(), k, 8)
            rr, r_pitch = _rows(residual.detach(), n, 8) if residual is not None else (None, n)
            _lib.check(lib.b200_linear_act_fwd(
                xr.data_ptr(), x_pitch, wr.data_ptr(), w_pitch, _ptr(b), ACTIVATIONS[activation], _ptr(rr), r_pitch, y.data_ptr(), _ptr(a),
                x.numel() // k, k, n, _DTYPES[x.dtype], _DTYPES[out_dtype], _stream()))
    return y, a


def linear_backward(dy: Tensor, x: Tensor | Checkpoint8 | None, weight: Tensor, pre: Tensor | None = None, activation: str | None = None,
                    bias: bool = True, needs: tuple[bool, bool] = (True, True), bias_dtype: torch.dtype = torch.float32
                    ) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    """``(dx, dw, db)`` of ``linear_forward`` for ``dy``, which has ``y``'s type; ``pre`` is what the forward pass saved (not needed without
    an activation), ``x`` its input or the 8-bit checkpoint of it (may be None where ``dw`` is not wanted).  ``needs`` says
    which of ``dx`` and ``dw`` are wanted, ``bias`` whether ``db`` is.  The gradient before the activation is rounded to the operands' type for the
    products, not for ``db``.  The residual's gradient is ``dy`` itself."""
    kept = x if isinstance(x, Checkpoint8) else None
    source = kept.values if kept else x
    _same_device(dy, source, weight, pre)
    if x is None:
        if needs[1]:
            raise ValueError("the weight's gradient wants x")
        k, n = _linear_sizes(dy.shape[:-1] + weight.shape[1:], weight.dtype, weight, activation)
        x_dtype, shape = weight.dtype, dy.shape[:-1] + (n,)
    else:
        k, n = _linear_sizes(source.shape, x.dtype, weight, activation)
        x_dtype, shape = x.dtype, source.shape[:-1] + (n,)
    if dy.shape != shape or dy.dtype not in (x_dtype, torch.float32):
        raise ValueError(f"dy must be {x_dtype} or float32 of shape {tuple(shape)}, got {dy.dtype} {tuple(dy.shape)}")
    if activation is not None and (pre is None or pre.shape != shape or pre.dtype != x_dtype):
        raise ValueError(f"pre must be {x_dtype} of shape {tuple(shape)}, got "
                         + ("None" if pre is None else f"{pre.dtype} {tuple(pre.shape)}"))
    bias_code = _code(bias_dtype, "the bias's gradient")
    with _on(dy.device):
        new = dict(device=dy.device)
        dx = torch.empty(shape[:-1] + (k,), dtype=x_dtype, **new) if needs[0] else None
        dw = torch.empty(n, k, dtype=x_dtype, **new) if needs[1] else None
        db = torch.empty(n, dtype=bias_dtype, **new) if bias else None
        if dx is None and dw is None and db is None:
            return None, None, None
        dyr, dy_pitch = _rows(dy.detach(), n, 8)
        g = _lib.LinearGrad(dy=_ptr(dyr), dy_pitch=dy_pitch, x_pitch=k, w_pitch=k, pre_pitch=n, dx=_ptr(dx), dw=_ptr(dw), db=_ptr(db),
                            rows=dy.numel() // n, k=k, n=n, act=ACTIVATIONS[activation], dtype=_DTYPES[x_dtype],
                            dy_dtype=_DTYPES[dy.dtype], db_dtype=bias_code)
        if kept:
            values, exponents = _kept(kept)
            g.values, g.exponents = values.data_ptr(), exponents.data_ptr()
        elif x is not None:
            xr, g.x_pitch = _rows(x.detach(), k, 8)
            g.x = xr.data_ptr()
        wr, g.w_pitch = _rows(weight.detach(), k, 8)
        g.w = wr.data_ptr()
        if activation is not None:
            pr, g.pre_pitch = _rows(pre.detach(), n, 8)
            g.pre = pr.data_ptr()
        size = lib.b200_linear_act_bwd_workspace_bytes(ctypes.byref(g))
        scratch = torch.empty(size, dtype=torch.uint8, **new) if size else None
        _lib.check(lib.b200_linear_act_bwd(ctypes.byref(g), _ptr(scratch), size, _stream()))
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
