"""Linear layers on microscaled 4-bit operands, for one weight and for a weight
per expert.  Both operands of every product are quantized along its contraction:

    y      = Q(x) Q(W)^T + bias           runs along the input index
    grad_x = Q(grad_y) Q(W^T)^T           runs along the output index
    grad_W = Q(grad_y^T) Q(x^T)^T         runs along the tokens
    grad_b = sum of grad_y over the tokens, from the unquantized gradient

The gradients pass the quantizers straight through.  What the backward needs of x
and W is kept as their 4-bit column forms, which the forward's one read of each
writes.
"""

from __future__ import annotations

from typing import Any

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import _native, hip_ops
from ..experts import ExpertRouting
from .mxfp4_matrix import MxFp4Weight, as_rows

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _check_input(x: torch.Tensor, in_dim: int) -> None:
    if x.dtype not in _DTYPES:
        raise NotImplementedError(f"the 4-bit linear takes bf16, fp16 or fp32 activations, got {x.dtype}")
    if x.ndim < 1 or x.shape[-1] != in_dim:
        raise ValueError(f"input {tuple(x.shape)} does not match weight input dim {in_dim}")
    if in_dim == 0:
        raise ValueError("the weight's input dim is zero")


def _differentiates() -> bool:
    """Whether a call may be recorded (or has to refuse a transform)."""
    return torch.is_grad_enabled() or torch._C._are_functorch_transforms_active() or forward_ad._current_level >= 0


def _weight_forms(weight: torch.Tensor | MxFp4Weight, needs_x: bool):
    """Row and column form of a weight, the latter where the input's gradient needs it."""
    if not isinstance(weight, MxFp4Weight):
        return hip_ops.mxfp4_quantize(as_rows(weight) if weight.ndim == 2 else weight.contiguous(), columns=needs_x)[:2]
    if needs_x and weight.transposed is None:
        raise RuntimeError(
            "a gradient for the input of a quantized weight needs its transposed form: "
            "quantize_mxfp4_weight(weight, transposed=True)"
        )
    return weight.matrix.pair, weight.transposed.pair if needs_x else None


def _linear_forward(x: torch.Tensor, weight: torch.Tensor | MxFp4Weight, bias: torch.Tensor | None, needs_x: bool, needs_w: bool):
    """The product, and the column forms of x and W that a backward needs."""
    x_rows, x_columns, _ = hip_ops.mxfp4_quantize(x, columns=needs_w)
    w_rows, w_columns = _weight_forms(weight, needs_x)
    out = hip_ops.mxfp4_gemm(x_rows, w_rows, x.dtype, bias=None if bias is None else bias.to(x.dtype).contiguous())
    return out, x_columns, w_columns


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, frozen: MxFp4Weight | None):
        needs_x, needs_w = ctx.needs_input_grad[0], frozen is None and ctx.needs_input_grad[1]
        out, x_columns, w_columns = _linear_forward(x, frozen or weight, bias, needs_x, needs_w)
        ctx.dtype, ctx.weight_dtype = x.dtype, None if frozen else weight.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.save_for_backward(*(x_columns or (None, None)), *(w_columns or (None, None)))
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad: torch.Tensor):
        x_data, x_scales, w_data, w_scales = ctx.saved_tensors
        needs_bias = ctx.bias_dtype is not None and ctx.needs_input_grad[2]
        grad = as_rows(grad)
        columns = x_data is not None or needs_bias
        g_rows, g_columns, sums = (None, None, None)
        if w_data is not None or columns:
            g_rows, g_columns, sums = hip_ops.mxfp4_quantize(grad, rows=w_data is not None, columns=columns, column_sums=needs_bias)
        grad_x = grad_w = grad_b = None
        if w_data is not None:
            grad_x = hip_ops.mxfp4_gemm(g_rows, (w_data, w_scales), ctx.dtype)
        if x_data is not None:
            grad_w = hip_ops.mxfp4_gemm(g_columns, (x_data, x_scales), ctx.weight_dtype)
        if needs_bias:
            grad_b = hip_ops.sum_runs(sums, ctx.bias_dtype)
        return grad_x, grad_w, grad_b, None


def mxfp4_linear(x: torch.Tensor, weight: torch.Tensor | MxFp4Weight, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ W.T + bias`` with both operands in microscaled 4-bit floats and fp32
    sums, rounded once to the type of ``x`` (bf16, fp16 or fp32).  ``weight``
    [out, in]: quantized within the call, with gradients for all three; an
    :class:`MxFp4Weight`: as it is, with gradients for ``x`` (if it has its
    transposed form) and ``bias``."""
    frozen = weight if isinstance(weight, MxFp4Weight) else None
    if len(weight.shape) != 2:
        raise ValueError(f"expected a weight [out, in], got {tuple(weight.shape)}")
    out_dim, in_dim = weight.shape
    _check_input(x, in_dim)
    if frozen is None and weight.dtype not in _DTYPES:
        raise NotImplementedError(f"the 4-bit linear takes bf16, fp16 or fp32 weights, got {weight.dtype}")
    if bias is not None and (tuple(bias.shape) != (out_dim,) or bias.dtype not in _DTYPES):
        raise ValueError(f"bias must be bf16, fp16 or fp32 [{out_dim}], got {bias.dtype} {tuple(bias.shape)}")
    if x.numel() == 0 or out_dim == 0:
        # no token or no output: autograd's own empty product keeps the graph
        dense = x.new_empty((out_dim, in_dim)) if frozen is not None else weight.to(x.dtype)
        return nn.functional.linear(x, dense, None if bias is None else bias.to(x.dtype))
    x_2d = as_rows(x if x.ndim == 2 else x.reshape(-1, in_dim))
    if _differentiates():
        out = _Linear.apply(x_2d, None if frozen else weight, bias, frozen)
    else:
        out = _linear_forward(x_2d, weight, bias, False, False)[0]
    return out if x.ndim == 2 else out.reshape(*x.shape[:-1], out_dim)


def _expert_forward(
    x: torch.Tensor, weight: torch.Tensor | MxFp4Weight, routing: ExpertRouting, sorted_rows: bool, needs_x: bool, needs_w: bool
):
    source = None if sorted_rows else routing.source
    x_rows = x_columns = None
    if needs_w:
        x_rows, x_columns = hip_ops.mxfp4_quantize_segments(
            x, routing.offsets, routing.padded_offsets, routing.padded_rows, choices=routing.rows, source=source,
            top_k=routing.top_k, rows=sorted_rows,
        )
    if x_rows is None:
        x_rows, _, _ = hip_ops.mxfp4_quantize(x)
    w_rows, w_columns = _weight_forms(weight, needs_x)
    out = hip_ops.mxfp4_gemm(
        x_rows, w_rows, x.dtype, mode=_native.MXFP4_ROWS, offsets=routing.offsets, source=source, top_k=routing.top_k,
        choices=routing.rows,
    )
    return out, x_columns, w_columns


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(
        ctx: Any, x: torch.Tensor, weight: torch.Tensor | None, routing: ExpertRouting, sorted_rows: bool, frozen: MxFp4Weight | None
    ):
        needs_x, needs_w = ctx.needs_input_grad[0], frozen is None and ctx.needs_input_grad[1]
        out, x_columns, w_columns = _expert_forward(x, frozen or weight, routing, sorted_rows, needs_x, needs_w)
        ctx.routing, ctx.sorted_rows = routing, sorted_rows
        ctx.dtype, ctx.weight_dtype = x.dtype, None if frozen else weight.dtype
        ctx.save_for_backward(*(x_columns or (None, None)), *(w_columns or (None, None)))
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad: torch.Tensor):
        x_data, x_scales, w_data, w_scales = ctx.saved_tensors
        routing = ctx.routing
        grad = as_rows(grad)
        grad_x = grad_w = g_rows = None
        if x_data is not None:
            g_rows, g_columns = hip_ops.mxfp4_quantize_segments(
                grad, routing.offsets, routing.padded_offsets, routing.padded_rows, choices=routing.rows, rows=w_data is not None,
            )
            grad_w = hip_ops.mxfp4_gemm(
                g_columns, (x_data, x_scales), ctx.weight_dtype, mode=_native.MXFP4_OVER_ROWS, offsets=routing.padded_offsets
            )
        elif w_data is not None:
            g_rows, _, _ = hip_ops.mxfp4_quantize(grad)
        if w_data is not None:
            grad_x = hip_ops.mxfp4_gemm(
                g_rows, (w_data, w_scales), ctx.dtype, mode=_native.MXFP4_ROWS, offsets=routing.offsets
            )
            if not ctx.sorted_rows:
                # The choices' gradients are rounded to the activation's type before they are added up in
                # fp32: half the bytes of fp32 rows, for an error of the size of the result's own rounding.
                grad_x = hip_ops.expert_combine(grad_x, routing.position)
        return grad_x, grad_w, None, None, None


def mxfp4_expert_linear(
    x: torch.Tensor, weight: torch.Tensor | MxFp4Weight, routing: ExpertRouting, *, sorted_rows: bool = False
) -> torch.Tensor:
    """Every expert's linear layer on its own rows: sorted row ``r`` of expert ``e``
    is ``x_r @ W_e.T``, [tokens * top_k, out]; rows of no expert are zero.  ``x`` is
    [tokens, in], each token's row read for all its experts, or with
    ``sorted_rows`` [tokens * top_k, in] in the order of ``routing``.  ``weight``
    [experts, out, in] as in :func:`mxfp4_linear`."""
    frozen = weight if isinstance(weight, MxFp4Weight) else None
    if len(weight.shape) != 3 or weight.shape[0] != routing.experts:
        raise ValueError(f"expected weights [{routing.experts}, out, in], got {tuple(weight.shape)}")
    _, out_dim, in_dim = weight.shape
    _check_input(x, in_dim)
    if frozen is None and weight.dtype not in _DTYPES:
        raise NotImplementedError(f"the 4-bit linear takes bf16, fp16 or fp32 weights, got {weight.dtype}")
    want = routing.rows if sorted_rows else routing.tokens
    if x.ndim != 2 or x.shape[0] != want:
        raise ValueError(f"x must be [{want}, {in_dim}], got {tuple(x.shape)}")
    if routing.rows == 0 or out_dim == 0:
        dense = x.new_empty((out_dim, in_dim)) if frozen is not None else weight[0].to(x.dtype)
        return nn.functional.linear(x.new_zeros((routing.rows, in_dim)) + 0 * x.sum(), dense)
    if _differentiates():
        return _ExpertLinear.apply(as_rows(x), None if frozen else weight, routing, sorted_rows, frozen)
    return _expert_forward(as_rows(x), weight, routing, sorted_rows, False, False)[0]


class FlexShardMxFp4Linear(nn.Linear):
    """``nn.Linear`` whose products run on microscaled 4-bit operands; the weight
    stays the (unsharded) bf16, fp16 or fp32 parameter."""

    @classmethod
    def from_float(cls, mod: nn.Linear) -> "FlexShardMxFp4Linear":
        with torch.device("meta"):
            new_mod = cls(mod.in_features, mod.out_features, bias=mod.bias is not None)
        new_mod.weight = mod.weight
        new_mod.bias = mod.bias
        new_mod.train(mod.training)
        return new_mod

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return mxfp4_linear(input, self.weight, self.bias)


def convert_to_flex_shard_mxfp4_linear(module: nn.Module, filter_fn=None) -> nn.Module:
    """Swap every ``nn.Linear`` below ``module`` that ``filter_fn(fqn, child)``
    accepts (all, when it is None) for a :class:`FlexShardMxFp4Linear` sharing its
    parameters."""
    _convert_children(module, "", filter_fn)
    return module


def _convert_children(parent: nn.Module, prefix: str, filter_fn) -> None:
    for name, child in list(parent.named_children()):
        fqn = f"{prefix}{name}"
        # (other quantized linears are subclasses and keep their own products)
        if type(child) is nn.Linear and (filter_fn is None or filter_fn(fqn, child)):
            setattr(parent, name, FlexShardMxFp4Linear.from_float(child))
        else:
            _convert_children(child, f"{fqn}.", filter_fn)


__all__ = ["FlexShardMxFp4Linear", "convert_to_flex_shard_mxfp4_linear", "mxfp4_expert_linear", "mxfp4_linear"]
