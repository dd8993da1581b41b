"""Root-mean-square norms ahead of the linears, with the residual's addition:

    h = x + residual,  y = h / sqrt(mean(h^2) + eps) * weight

:func:`rms_norm` gives y in the type of ``x``, :func:`rms_norm_fp8` in the 8 bits that
the blockwise FP8 linears multiply (``flex_shard_amd.blockwise_fp8``), so that no linear
quantizes it again.  Both also return h where there is a residual: the stream that the
next layer adds to.  The norm is that of h as it is kept, rounded to the residual's type.
"""

from __future__ import annotations

from functools import partial
from typing import Any

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import hip_ops
from ..blockwise_fp8.fp8_activation import Fp8Activation
from ..experts import differentiates

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
# Of a module that names none: torch's own takes that of the type it computes in, also for bf16 and fp16
# rows.  (Of rows of 0.01 the norm with bf16's would be 0.11, not 1.)
_EPS = torch.finfo(torch.float32).eps


def _as_rows(t: torch.Tensor) -> torch.Tensor:
    """Contiguous rows [..., cols], or a matrix of contiguous rows that do not
    overlap; a copy if need be."""
    if t.is_contiguous() or (
        t.ndim == 2 and (t.shape[1] <= 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1])
    ):
        return t
    return t.contiguous()


def _check(x: torch.Tensor, weight: torch.Tensor | None, eps: float, residual: torch.Tensor | None) -> None:
    """For a call without rows; any other one is checked with its operands."""
    if x.dtype not in _DTYPES:
        raise NotImplementedError(f"the norm takes bf16, fp16 or fp32 rows, got {x.dtype}")
    if x.ndim < 1 or x.shape[-1] == 0:
        raise ValueError(f"expected rows [..., cols], got {tuple(x.shape)}")
    if weight is not None and (tuple(weight.shape) != (x.shape[-1],) or weight.dtype not in _DTYPES):
        raise ValueError(f"weight must be bf16, fp16 or fp32 [{x.shape[-1]}], got {weight.dtype} {tuple(weight.shape)}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual must be {tuple(x.shape)}, got {tuple(residual.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise NotImplementedError(f"a residual is of the type of x ({x.dtype}) or fp32, got {residual.dtype}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")


def _carrier(shape, device: torch.device) -> torch.Tensor:
    # (of one element, and not an expanded view of it: autograd would go back through its strides)
    return torch.empty_strided(shape, (0,) * len(shape), dtype=torch.bfloat16, device=device)


class _Norm(torch.autograd.Function):
    """``(y, total)``; in 8 bits y is the carrier, and ``kept`` gets the bytes, the
    scales and what the token runs are made of."""

    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor | None, eps: float, kept: list | None):
        out, total, rstd = hip_ops.rms_norm(x, weight, eps, residual, fp8=kept is not None, keep_rstd=True)
        normed = x if total is None else total
        if kept is not None:
            kept += (*out, normed, rstd)
            out = _carrier(x.shape, x.device)
        ctx.save_for_backward(normed, weight, rstd)
        # what the backward's thread need not find out again
        cols, types, x_dtype = x.shape[-1], hip_ops.FLOAT_CODES, x.dtype
        codes = types[out.dtype], types[normed.dtype], types[x_dtype], 0 if weight is None else types[weight.dtype]
        ctx.call = x_dtype, x.numel() // cols, cols, codes
        ctx.kept = x.get_device(), normed.nbytes, normed.dtype, 0 if weight is None else weight.nbytes, None if weight is None else weight.dtype
        ctx.set_materialize_grads(False)
        return out, total

    @staticmethod
    def backward(ctx: Any, grad: torch.Tensor | None, grad_total: torch.Tensor | None):
        # (recorded only for a second differentiation, which the wrapper refuses: 3 us of the backward's thread else)
        return (_norm_backward_once if torch.is_grad_enabled() else _norm_backward)(ctx, grad, grad_total)


def _norm_backward(ctx: Any, grad: torch.Tensor | None, grad_total: torch.Tensor | None):
    x_dtype, rows, cols, codes = ctx.call
    needs_x, needs_residual, needs_weight, _, _ = ctx.needs_input_grad
    if grad is None:  # the stream alone was used
        if grad_total is None:
            return None, None, None, None, None
        return grad_total.to(x_dtype) if needs_x else None, grad_total if needs_residual else None, None, None, None
    normed, weight, rstd = ctx.saved_tensors
    ldg = ldh = ldt = cols
    if not grad.is_contiguous():
        grad = _as_rows(grad)
        ldg = cols if grad.is_contiguous() else grad.stride(0)
    if not normed.is_contiguous():
        normed = _as_rows(normed) if normed.shape[-1] == cols else normed.contiguous()
        ldh = cols if normed.is_contiguous() else normed.stride(0)
    if grad_total is not None and not grad_total.is_contiguous():
        grad_total = _as_rows(grad_total)
        ldt = cols if grad_total.is_contiguous() else grad_total.stride(0)
    # (autograd answers for the gradients; hooks on saved tensors may give back others than were kept)
    index, nbytes, dtype, weight_nbytes, weight_dtype = ctx.kept
    if (
        normed.get_device() != index or normed.nbytes != nbytes or normed.dtype is not dtype or rstd.get_device() != index
        or rstd.dtype is not torch.float32 or rstd.nbytes != 4 * rows or not rstd.is_contiguous()
    ) or (
        weight is not None and (
            weight.get_device() != index or weight.nbytes != weight_nbytes or weight.dtype is not weight_dtype or not weight.is_contiguous()
        )
    ):
        raise RuntimeError("a hook on saved tensors gave back other tensors than the norm kept")
    grad_x, grad_residual, grad_weight = hip_ops.rms_norm_backward_checked(
        grad, normed, weight, rstd, x_dtype, grad_total, (rows, cols, ldg, ldh, ldt), codes, needs_x, needs_residual, needs_weight
    )
    return grad_x, grad_residual, grad_weight, None, None


_norm_backward_once = once_differentiable(_norm_backward)


def rms_norm(
    x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6, *, residual: torch.Tensor | None = None
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """The norm of the rows of ``x`` [..., cols] (bf16, fp16 or fp32), in its type,
    times ``weight`` [cols] (any of these types, or None).  With ``residual``, of the
    shape of ``x`` and its type or fp32, ``(norm of x + residual, x + residual)``, the sum in
    the residual's type.  Statistics in fp32, every output rounded once; differentiable.
    A row's bits are the same on every run, but a call of more than 512 rows of 2049 to 8192 columns
    adds up a row in another order than one of fewer: a prompt's row and the same one alone may
    differ by a rounding."""
    if x.numel() == 0:  # no rows: torch's own empty products keep the graph
        _check(x, weight, eps, residual)
        total = x if residual is None else x.to(residual.dtype) + residual
        y = (total if weight is None else total * weight).to(x.dtype)
        return y if residual is None else (y, total)
    x = _as_rows(x)
    stream = None if residual is None else _as_rows(residual)
    weight = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    if differentiates(x, stream, weight):
        y, total = _Norm.apply(x, stream, weight, eps, None)
    else:
        y, total, _ = hip_ops.rms_norm(x, weight, eps, stream)
    return y if residual is None else (y, total)


def _version(t: torch.Tensor | None) -> int:
    return 0 if t is None or t.is_inference() else t._version


def _token_runs(normed, weight, rstd, versions: tuple[int, int]) -> tuple[torch.Tensor, torch.Tensor]:
    if versions != (_version(normed), _version(weight)):
        raise RuntimeError("what an 8-bit norm was made of was changed in place before a weight gradient's form of it was made")
    return hip_ops.rms_norm_token_runs(normed, weight, rstd)


def rms_norm_fp8(
    x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6, *, residual: torch.Tensor | None = None
) -> Fp8Activation | tuple[Fp8Activation, torch.Tensor]:
    """:func:`rms_norm`, its output rounded to bf16 and quantized like the
    activations of the blockwise FP8 linears, which take it as it is."""
    x = _as_rows(x)
    stream = None if residual is None else _as_rows(residual)
    weight = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    if x.numel() == 0:
        y = rms_norm(x, weight, eps, residual=residual)
        carrier, total = (y, None) if residual is None else y
        (q, scales), _, rstd = hip_ops.rms_norm(x, None, eps, fp8=True, keep_rstd=True)
        normed, carrier = x, carrier.to(torch.bfloat16)
    elif differentiates(x, stream, weight):
        kept: list = []
        carrier, total = _Norm.apply(x, stream, weight, eps, kept)
        q, scales, normed, rstd = kept
    else:
        (q, scales), total, rstd = hip_ops.rms_norm(x, weight, eps, stream, fp8=True, keep_rstd=True)
        normed, carrier = x if total is None else total, _carrier(x.shape, x.device)
    if weight is not None and torch.is_grad_enabled():
        # The token runs are made when a linear asks for them, and by then the weight's
        # bucket may be resharded, or an optimizer have been at it.
        weight = weight.detach().clone()
    activation = Fp8Activation(
        q, scales, carrier, partial(_token_runs, normed, weight, rstd, (_version(normed), _version(weight))),
        (normed, rstd) if weight is None else (normed, rstd, weight),
    )
    return activation if residual is None else (activation, total)


class FlexShardRMSNorm(nn.RMSNorm):
    """``nn.RMSNorm`` over the last dimension on the kernels here.  ``forward(x,
    residual)`` adds first and returns the sum too; with ``fp8`` the output is an
    :class:`~flex_shard_amd.blockwise_fp8.Fp8Activation`.  ``eps`` None is fp32's."""

    @classmethod
    def from_float(cls, mod: nn.RMSNorm) -> "FlexShardRMSNorm":
        if len(mod.normalized_shape) != 1:
            raise NotImplementedError(f"the norm is over the last dimension, got {tuple(mod.normalized_shape)}")
        new_mod = cls(mod.normalized_shape, eps=mod.eps, elementwise_affine=mod.elementwise_affine, device="meta")
        new_mod.weight = mod.weight
        new_mod.train(mod.training)
        return new_mod

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, *, fp8: bool = False):
        if len(self.normalized_shape) != 1 or x.shape[-1:] != tuple(self.normalized_shape):
            raise ValueError(f"the norm is over a last dimension {tuple(self.normalized_shape)}, got {tuple(x.shape)}")
        eps = _EPS if self.eps is None else self.eps
        return (rms_norm_fp8 if fp8 else rms_norm)(x, self.weight, eps, residual=residual)


def convert_to_flex_shard_rms_norm(module: nn.Module, filter_fn=None) -> nn.Module:
    """Swap every ``nn.RMSNorm`` over one dimension below ``module`` that
    ``filter_fn(fqn, child)`` accepts (all, when it is None) for a
    :class:`FlexShardRMSNorm` sharing its weight; one that has several names for the
    same module under each of them."""
    _convert_children(module, "", filter_fn, {})
    return module


def _convert_children(parent: nn.Module, prefix: str, filter_fn, converted: dict[nn.Module, nn.Module]) -> None:
    for name, child in list(parent._modules.items()):  # (named_children leaves second names out)
        if child is None:
            continue
        fqn = f"{prefix}{name}"
        if type(child) is nn.RMSNorm and len(child.normalized_shape) == 1 and (filter_fn is None or filter_fn(fqn, child)):
            if child not in converted:
                converted[child] = FlexShardRMSNorm.from_float(child)
            setattr(parent, name, converted[child])
        else:
            _convert_children(child, f"{fqn}.", filter_fn, converted)


__all__ = ["FlexShardRMSNorm", "convert_to_flex_shard_rms_norm", "rms_norm", "rms_norm_fp8"]
