"""Operators for training a model next to the inference kernels: LayerNorm and the linear layer with their gradients, and
activation checkpoints in 8 bits that the backward passes take in the activation's place.

Three levels, each on the current stream of the tensors' device:

- ``layer_norm_forward`` / ``layer_norm_backward``, ``linear_forward`` / ``linear_backward``, ``checkpoint8``: the passes themselves;
- ``layer_norm`` and ``linear``: the same as differentiable functions (``checkpoint=True`` keeps ``x`` in 8 bits for backward), in
  reverse mode and once;
- ``LayerNorm`` and ``Linear``: modules with the parameters of their ``torch.nn`` namesakes.

Scratch comes from torch's caching allocator call by call, so calls may be captured into CUDA graphs and may run at the same
time on several streams.  The order of every sum goes by the sizes alone: equal calls give equal bits.  Bad arguments raise
``ValueError`` before anything is launched, tensors without memory of their own (DTensor and other wrappers) among them.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from . import _lib

try:
    from . import _training
except ImportError as error:
    raise ImportError(f"bioemu2_b200/_training.so has not been built, or was built for another torch (run `python __graft_entry__.py` at the "
                      f"repository root): {error}") from error

_training.bind({name: ctypes.cast(getattr(_lib.lib, name), ctypes.c_void_p).value for name in
                ("b200_layer_norm_save_fwd", "b200_layer_norm_bwd_workspace_bytes", "b200_layer_norm_bwd", "b200_checkpoint8_fwd",
                 "b200_checkpoint8_restore", "b200_linear_act_fwd", "b200_linear_act_bwd_workspace_bytes", "b200_linear_act_bwd")}, _lib.check)

GROUP = 32          # neighbours in a row that share a power of two in an 8-bit checkpoint
MAX_COLS = 8192     # of a LayerNorm row
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _activation(name: str | None) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(a for a in ACTIVATIONS if a)} or None, got {name!r}")
    return ACTIVATIONS[name]


class Checkpoint8(NamedTuple):
    """An activation in 8 bits: ``values`` (``float8_e4m3fn``, the activation's shape) times ``2 ** (exponents - 127)``, one
    exponent (``uint8``) for each 32 neighbours along the last axis, the last of them possibly fewer.  A group's exponent is the
    least, from -127 up, with which its largest finite magnitude is at most 448 times the power; infinities are kept as NaN.
    Finite values stay finite: one that rounds past the largest of the type it comes back in is that largest value.
    ``dtype`` is the activation's type."""

    values: Tensor
    exponents: Tensor
    dtype: torch.dtype

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    def restore(self, dtype: torch.dtype | None = None) -> Tensor:
        """The activation as it was kept, rounded to ``dtype`` (the activation's own)."""
        return _training.restore8(self.values, self.exponents, dtype or self.dtype)


def checkpoint8(x: Tensor) -> Checkpoint8:
    """``x`` (fp32, bf16 or fp16, rows of 1 to 2^31 - 1 columns) in 8 bits: 1 + 1/32 bytes an element."""
    return Checkpoint8(*_training.checkpoint8(x), x.dtype)


def _differentiated(x: Tensor, weight: Tensor | None, bias: Tensor | None, residual: Tensor | None = None) -> bool:
    """Whether backward will ask for a gradient of a call with these inputs.  Tangents of forward-mode differentiation ask for one that
    is not there; without a word the result would have none, and so a derivative of zero."""
    if _training.has_tangent(x, weight, bias, residual):
        raise NotImplementedError("layer_norm and linear have no forward-mode derivative")
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual))


# ---------------------------------------------------------------------------------------------------------------------------
# LayerNorm
# ---------------------------------------------------------------------------------------------------------------------------
def layer_norm_forward(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5,
                       out_dtype: torch.dtype | None = None, checkpoint: bool = False
                       ) -> tuple[Tensor, Tensor, Tensor, Checkpoint8 | None]:
    """``(y, mean, rstd, kept)``: ``y = (x - mean) * rstd * weight + bias`` over the last axis, fp32 statistics of shape
    ``x.shape[:-1]``, and with ``checkpoint`` ``x`` in 8 bits, written by the same pass.  An fp32 ``x`` may have ``y`` in any of the
    three types (``out_dtype``)."""
    y, mean, rstd, values, exponents = _training.layer_norm_forward(x, weight, bias, eps, out_dtype, checkpoint)
    return y, mean, rstd, Checkpoint8(values, exponents, x.dtype) if checkpoint else None


def layer_norm_backward(dy: Tensor, x: Tensor | Checkpoint8, mean: Tensor, rstd: Tensor, weight: Tensor | None = None,
                        needs: tuple[bool, bool, bool] | None = None, grad_dtype: torch.dtype | None = None
                        ) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    """``(dx, dw, db)`` from the forward pass's ``mean`` and ``rstd`` and either its ``x`` or the 8-bit checkpoint of it (``dx`` then
    has the type of what was kept).  ``needs`` says which of the three are wanted: all with a weight, ``dx`` alone without one.
    ``dw`` and ``db`` have ``grad_dtype``, by default the weight's type (float32 without one)."""
    if isinstance(x, Checkpoint8):
        return _training.layer_norm_backward(dy, x.values, x.exponents, x.dtype, mean, rstd, weight, needs, grad_dtype)
    return _training.layer_norm_backward(dy, x, None, None, mean, rstd, weight, needs, grad_dtype)


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
        types = {t for t in (weight.dtype if weight is not None else None, ctx.bias_dtype) if t is not None}
        # parameters of two types: the fp32 sums, each rounded to its own
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight, needs, types.pop() if len(types) == 1 else torch.float32)
        return dx, dw if dw is None else dw.to(weight.dtype), db if db is None else db.to(ctx.bias_dtype), None, None, None


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, eps: float = 1e-5,
               out_dtype: torch.dtype | None = None, checkpoint: bool = False) -> Tensor:
    """``layer_norm_forward``'s ``y`` as a differentiable function; ``checkpoint`` keeps ``x`` in 8 bits for the backward pass."""
    if _differentiated(x, weight, bias):
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
def linear_forward(x: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = None,
                   residual: Tensor | None = None, out_dtype: torch.dtype | None = None, save: bool | torch.dtype = False
                   ) -> tuple[Tensor, Tensor | None]:
    """``(y, a)``: ``y = act(a) + residual`` with ``a = x @ weight.T + bias``.  ``x[..., in]`` and ``weight[out, in]`` are both bf16 or both
    fp16, ``in`` and ``out`` multiples of 8, at most 2^24.  ``y`` has ``out_dtype``, the operands' type or fp32: by default the residual's,
    which is ``y``'s, or the operands'.  ``gelu`` is off by 1e-7 of its argument at most, which far below zero leaves it few digits.
    ``a`` is returned for the backward pass with ``save``: rounded to the operands' type, or with ``save=torch.float32`` as it is, for gradients without that rounding (None without an activation, which needs none)."""
    save_dtype = save if isinstance(save, torch.dtype) else x.dtype if save else None
    return _training.linear_forward(x, weight, bias, _activation(activation), residual, out_dtype, save_dtype)


def linear_backward(dy: Tensor, x: Tensor | Checkpoint8 | None, weight: Tensor, pre: Tensor | None = None, activation: str | None = None,
                    bias: bool = True, needs: tuple[bool, bool] = (True, True), bias_dtype: torch.dtype = torch.float32
                    ) -> tuple[Tensor | None, Tensor | None, Tensor | None]:
    """``(dx, dw, db)`` of ``linear_forward`` for ``dy``, which has ``y``'s type; ``pre`` is what the forward pass saved (not needed without
    an activation), ``x`` its input or the 8-bit checkpoint of it (may be None where ``dw`` is not wanted).  ``needs`` says which of
    ``dx`` and ``dw`` are wanted, ``bias`` whether ``db`` is.  The gradient before the activation is rounded to the operands' type for the
    products, not for ``db``.  The residual's gradient is ``dy`` itself."""
    exponents = dtype = None
    if isinstance(x, Checkpoint8):
        x, exponents, dtype = x
    return _training.linear_backward(dy, x, exponents, dtype, weight, pre, _activation(activation), needs[0], needs[1],
                                     bias_dtype if bias else None)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation, residual, out_dtype, checkpoint, save_dtype):
        y, pre = linear_forward(x, weight, bias, activation, residual, out_dtype, any(ctx.needs_input_grad[:3]) and (save_dtype or True))
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
        return dx, dw, db, None, dy if ctx.needs_input_grad[4] else None, None, None, None


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str | None = None, residual: Tensor | None = None,
           out_dtype: torch.dtype | None = None, checkpoint: bool = False, save_dtype: torch.dtype | None = None) -> Tensor:
    """``linear_forward``'s ``y`` as a differentiable function; ``checkpoint`` keeps ``x`` in 8 bits for the weight's gradient.  The value
    before an activation is kept in ``save_dtype``: the operands' type (default), or float32 for slopes without that rounding (2^-9 of
    the value in bf16, which is what the bias's fp32 sum then loses)."""
    if save_dtype not in (None, torch.float32, x.dtype):
        raise ValueError(f"the value before the activation is saved as {x.dtype} like x or float32, not as {save_dtype}")
    if _differentiated(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, activation, residual, out_dtype, checkpoint, save_dtype)
    return linear_forward(x, weight, bias, activation, residual, out_dtype)[0]


class Linear(nn.Linear):
    """``torch.nn.Linear`` with an activation and a residual in the product's epilogue, on bf16 or fp16 inputs; parameters of another
    type (fp32 masters) are rounded to the input's type at each call.  ``out_dtype``, ``checkpoint`` and ``save_dtype`` are ``linear``'s."""

    save_dtype: torch.dtype | None = None  # of modules pickled without it

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: str | None = None,
                 out_dtype: torch.dtype | None = None, checkpoint: bool = False, device=None, dtype=None,
                 save_dtype: torch.dtype | None = None) -> None:
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        _activation(activation)
        if in_features % 8 or out_features % 8 or in_features < 1 or out_features < 1:
            raise ValueError(f"in_features={in_features} and out_features={out_features} must be positive multiples of 8")
        self.activation, self.out_dtype, self.checkpoint, self.save_dtype = activation, out_dtype, checkpoint, save_dtype

    def forward(self, x: Tensor, residual: Tensor | None = None) -> Tensor:
        weight = self.weight if self.weight.dtype == x.dtype else self.weight.to(x.dtype)
        return linear(x, weight, self.bias, self.activation, residual, self.out_dtype, self.checkpoint, self.save_dtype)
