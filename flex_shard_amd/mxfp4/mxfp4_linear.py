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
from torch.autograd.function import once_differentiable

from .. import _native, hip_ops
from ..experts import ExpertRouting, check_routing, differentiates
from ..hip_ops import MxFp4Matrix
from .mxfp4_matrix import MxFp4Weight, as_rows

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _check_input(x: torch.Tensor, in_dim: int) -> None:
    if x.dtype not in _DTYPES:
        raise NotImplementedError(f"the 4-bit linear takes bf16, fp16 or fp32 activations, got {x.dtype}")
    if x.ndim < 1 or x.shape[-1] != in_dim:
        raise ValueError(f"input {tuple(x.shape)} does not match weight input dim {in_dim}")
    if in_dim == 0:
        raise ValueError("the weight's input dim is zero")


def _weight_forms(weight: torch.Tensor | MxFp4Weight, needs_x: bool):
    """Row and column form of a weight, the latter where the input's gradient needs it."""
    if not isinstance(weight, MxFp4Weight):
        return hip_ops.mxfp4_quantize(as_rows(weight) if weight.ndim == 2 else weight.contiguous(), columns=needs_x)[:2]
    if needs_x and weight.transposed is None:
        raise RuntimeError(
            "a gradient for the input of a quantized weight needs its transposed form: "
            "quantize_mxfp4_weight(weight, transposed=True)"
        )
    return weight.matrix, weight.transposed if needs_x else None


def _bias_for(x: torch.Tensor, bias: torch.Tensor | None) -> torch.Tensor | None:
    """The bias as the product's epilogue adds it, before the one rounding: of the
    activation's type or fp32, which any other becomes without a rounding."""
    if bias is None:
        return bias
    return (bias if bias.dtype == x.dtype else bias.float()).contiguous()


def _keep(ctx: Any, x_columns: MxFp4Matrix | None, w_columns: MxFp4Matrix | None) -> None:
    """Save the column forms that the backward reads."""
    ctx.forms = [None if form is None else (form.rows, form.cols) for form in (x_columns, w_columns)]
    ctx.save_for_backward(*[None if form is None else form.buffer for form in (x_columns, w_columns)])


def _kept(ctx: Any) -> list[MxFp4Matrix | None]:
    return [None if size is None else MxFp4Matrix(buffer, *size) for buffer, size in zip(ctx.saved_tensors, ctx.forms)]


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, frozen: MxFp4Weight | None):
        needs_x, needs_w = ctx.needs_input_grad[0], frozen is None and ctx.needs_input_grad[1]
        w_rows, w_columns = _weight_forms(frozen or weight, needs_x)
        x_columns = None
        if needs_w:
            x_rows, x_columns, _ = hip_ops.mxfp4_quantize(x, columns=True)
            out = hip_ops.mxfp4_gemm(x_rows, w_rows, x.dtype, bias=_bias_for(x, bias))
        else:
            out = hip_ops.mxfp4_linear(x, w_rows, _bias_for(x, bias))
        ctx.dtype, ctx.weight_dtype = x.dtype, None if frozen else weight.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        _keep(ctx, x_columns, w_columns)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad: torch.Tensor):
        x_columns, w_columns = _kept(ctx)
        needs_bias = ctx.bias_dtype is not None and ctx.needs_input_grad[2]
        columns = x_columns is not None or needs_bias
        grad_x = grad_w = grad_b = None
        if w_columns is not None or columns:
            g_rows, g_columns, sums = hip_ops.mxfp4_quantize(
                as_rows(grad), rows=w_columns is not None, columns=columns, column_sums=needs_bias
            )
        if w_columns is not None:
            grad_x = hip_ops.mxfp4_gemm(g_rows, w_columns, ctx.dtype)
        if x_columns is not None:
            grad_w = hip_ops.mxfp4_gemm(g_columns, x_columns, ctx.weight_dtype)
        if needs_bias:
            grad_b = hip_ops.sum_runs(sums, ctx.bias_dtype)
        return grad_x, grad_w, grad_b, None


def mxfp4_linear(x: torch.Tensor, weight: torch.Tensor | MxFp4Weight, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ W.T + bias`` with both operands in microscaled 4-bit floats and fp32
    sums, rounded once to the type of ``x`` (bf16, fp16 or fp32); a bias of another
    of these types is added unrounded.  ``weight``
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
    if differentiates(x_2d, None if frozen else weight, bias):
        out = _Linear.apply(x_2d, None if frozen else weight, bias, frozen)
    else:
        out = hip_ops.mxfp4_linear(x_2d, _weight_forms(weight, False)[0], _bias_for(x, bias))
    return out if x.ndim == 2 else out.reshape(*x.shape[:-1], out_dim)


def _expert_forward(x: torch.Tensor, w_rows: MxFp4Matrix, routing: ExpertRouting, sorted_rows: bool) -> torch.Tensor:
    _, source, offsets, _ = routing.pointers()
    return hip_ops.mxfp4_expert_linear(
        x, w_rows, routing.experts, routing.rows, routing.top_k, offsets, None if sorted_rows else source
    )


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(
        ctx: Any, x: torch.Tensor, weight: torch.Tensor | None, routing: ExpertRouting, sorted_rows: bool, frozen: MxFp4Weight | None
    ):
        needs_x, needs_w = ctx.needs_input_grad[0], frozen is None and ctx.needs_input_grad[1]
        w_rows, w_columns = _weight_forms(frozen or weight, needs_x)
        x_rows = x_columns = None
        if needs_w:
            x_rows, x_columns = hip_ops.mxfp4_quantize_segments(
                x, routing.offsets, routing.padded_offsets, routing.padded_rows, choices=routing.rows,
                source=None if sorted_rows else routing.source, top_k=routing.top_k, rows=sorted_rows,
            )
        if x_rows is not None:
            out = hip_ops.mxfp4_gemm(x_rows, w_rows, x.dtype, mode=_native.MXFP4_ROWS, offsets=routing.offsets)
        else:
            out = _expert_forward(x, w_rows, routing, sorted_rows)
        ctx.routing, ctx.sorted_rows = routing, sorted_rows
        ctx.dtype, ctx.weight_dtype = x.dtype, None if frozen else weight.dtype
        _keep(ctx, x_columns, w_columns)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad: torch.Tensor):
        x_columns, w_columns = _kept(ctx)
        routing = ctx.routing
        grad = as_rows(grad)
        grad_x = grad_w = g_rows = None
        if x_columns is not None:
            g_rows, g_columns = hip_ops.mxfp4_quantize_segments(
                grad, routing.offsets, routing.padded_offsets, routing.padded_rows, choices=routing.rows, rows=w_columns is not None,
            )
            grad_w = hip_ops.mxfp4_gemm(
                g_columns, x_columns, ctx.weight_dtype, mode=_native.MXFP4_OVER_ROWS, offsets=routing.padded_offsets
            )
        elif w_columns is not None:
            g_rows, _, _ = hip_ops.mxfp4_quantize(grad)
        if w_columns is not None:
            # The parts of a token that several experts have are added up in fp32 and rounded once.  In 16 bits they
            # would be half the bytes (a training step of 4096 tokens, 8 of 32 experts [2048, 7168] each: 1690 us for
            # 1850), but rounded twice, and fp16 parts can pass its range where their sum does not.
            parts = torch.float32 if not ctx.sorted_rows and routing.top_k > 1 else ctx.dtype
            grad_x = hip_ops.mxfp4_gemm(g_rows, w_columns, parts, mode=_native.MXFP4_ROWS, offsets=routing.offsets)
            if not ctx.sorted_rows:
                grad_x = hip_ops.expert_combine_at(grad_x, routing.pointers()[0], routing.tokens, routing.top_k, dtype=ctx.dtype)
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
    check_routing(routing, x)
    x = as_rows(x)
    if differentiates(x, None if frozen else weight):
        if x.requires_grad and not sorted_rows and routing.top_k > _native.MAX_CHOICES:
            raise NotImplementedError(
                f"a gradient for the tokens adds up at most {_native.MAX_CHOICES} choices each, got {routing.top_k} (rows in sorted order, "
                "sorted_rows=True, have no such limit)"
            )
        return _ExpertLinear.apply(x, None if frozen else weight, routing, sorted_rows, frozen)
    return _expert_forward(x, _weight_forms(weight, False)[0], routing, sorted_rows)


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
