"""Tokens sorted by expert and back.

A router gives every token ``top_k`` experts and weights.  :func:`route_tokens`
sorts the choices by expert, :func:`dispatch_tokens` gathers the tokens' rows in
that order, and :func:`combine_tokens` brings the experts' rows back, weighted.
``flex_shard_amd.mxfp4.mxfp4_expert_linear`` multiplies the rows in between.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Any

import torch
from torch.autograd.function import once_differentiable

from .. import hip_ops


@dataclass(frozen=True)
class ExpertRouting:
    """The choices [tokens, top_k] of a router in stable order by expert.  There
    are tokens * top_k sorted rows; rows from ``offsets[-1]`` on belong to choices
    of no expert here, hold nothing, and are zero wherever they are written."""

    experts: int
    #: [tokens, top_k] int32: the sorted row of each choice, -1 for no expert here
    position: torch.Tensor
    #: [experts + 1] int32: expert ``e`` has rows ``offsets[e]`` to ``offsets[e + 1]``
    offsets: torch.Tensor
    #: [tokens * top_k] int32: the choice ``t * top_k + j`` of each sorted row, -1 behind the last
    source: torch.Tensor
    #: [experts + 1] int32: the segments, each rounded up to 256 rows (a product over an expert's rows)
    padded_offsets: torch.Tensor

    @property
    def tokens(self) -> int:
        return self.position.shape[0]

    @property
    def top_k(self) -> int:
        return self.position.shape[1]

    @property
    def rows(self) -> int:
        return self.source.numel()

    @property
    def padded_rows(self) -> int:
        """Rows that the padded segments take at most."""
        return (self.rows + 255 * min(self.experts, self.rows)) // 256 * 256


def route_tokens(expert_ids: torch.Tensor, experts: int) -> ExpertRouting:
    """Sort the choices ``expert_ids`` [tokens, top_k] (int64 or int32) by expert.
    An id outside [0, experts) -- an expert of another rank, a choice dropped -- is
    a choice of no expert here.  Nothing waits for the GPU."""
    if expert_ids.ndim != 2 or expert_ids.shape[1] == 0:
        raise ValueError(f"expert_ids must be [tokens, top_k], got {tuple(expert_ids.shape)}")
    if experts <= 0:
        raise ValueError(f"at least one expert, got {experts}")
    return ExpertRouting(experts, *hip_ops.expert_route(expert_ids.contiguous(), experts))


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, routing: ExpertRouting) -> torch.Tensor:
        ctx.routing = routing
        return hip_ops.expert_dispatch(x.contiguous(), routing.position, routing.offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad: torch.Tensor):
        return hip_ops.expert_combine(grad.contiguous(), ctx.routing.position), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, rows: torch.Tensor, weights: torch.Tensor, routing: ExpertRouting) -> torch.Tensor:
        rows, weights = rows.contiguous(), weights.contiguous()
        ctx.routing = routing
        ctx.save_for_backward(rows, weights)
        return hip_ops.expert_combine(rows, routing.position, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad: torch.Tensor):
        rows, weights = ctx.saved_tensors
        return (*hip_ops.expert_combine_backward(grad.contiguous(), rows, ctx.routing.position, ctx.routing.offsets, weights), None)


def dispatch_tokens(x: torch.Tensor, routing: ExpertRouting) -> torch.Tensor:
    """The tokens' rows [tokens, width] (bf16, fp16 or fp32) gathered into sorted
    rows [tokens * top_k, width], differentiable: a token's gradient is the sum of
    its rows' gradients, in fp32 in the order of its choices."""
    if x.ndim != 2 or x.shape[0] != routing.tokens:
        raise ValueError(f"x must be [{routing.tokens}, width], got {tuple(x.shape)}")
    return _Dispatch.apply(x, routing)


def combine_tokens(rows: torch.Tensor, routing: ExpertRouting, weights: torch.Tensor) -> torch.Tensor:
    """``out[t] = sum_j weights[t, j] * rows[position[t, j]]`` for sorted rows
    [tokens * top_k, width], differentiable in both; fp32 sums in the order of j,
    rounded once.  A token none of whose experts are here gets zeros."""
    if rows.ndim != 2 or rows.shape[0] != routing.rows:
        raise ValueError(f"rows must be [{routing.rows}, width], got {tuple(rows.shape)}")
    if weights.shape != routing.position.shape:
        raise ValueError(f"weights must be {tuple(routing.position.shape)}, got {tuple(weights.shape)}")
    return _Combine.apply(rows, weights, routing)


__all__ = ["ExpertRouting", "combine_tokens", "dispatch_tokens", "route_tokens"]
