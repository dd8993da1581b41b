"""Tokens sorted by expert and back.

A router gives every token ``top_k`` experts and weights.  :func:`route_tokens`
sorts the choices by expert, :func:`dispatch_tokens` gathers the tokens' rows in
that order, and :func:`combine_tokens` brings the experts' rows back, weighted.
``flex_shard_amd.mxfp4.mxfp4_expert_linear`` multiplies the rows in between.
"""

from __future__ import annotations

from typing import Any

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import hip_ops


class ExpertRouting:
    """The choices [tokens, top_k] of a router in stable order by expert.  There
    are tokens * top_k sorted rows; rows from ``offsets[-1]`` on belong to choices
    of no expert here, hold nothing, and are zero wherever they are written.

    ``position`` [tokens, top_k]: the sorted row of each choice, -1 for no expert
    here.  ``offsets`` [experts + 1]: expert ``e`` has rows ``offsets[e]`` to
    ``offsets[e + 1]``.  ``source`` [tokens * top_k]: the choice ``t * top_k + j`` of
    each sorted row, -1 behind the last.  ``padded_offsets`` [experts + 1]: the
    segments, each rounded up to 256 rows (a product over an expert's rows).  All
    int32, behind one another in one buffer."""

    __slots__ = ("experts", "tokens", "top_k", "rows", "buffer")

    def __init__(
        self, experts: int, position: torch.Tensor, offsets: torch.Tensor, source: torch.Tensor, padded_offsets: torch.Tensor
    ) -> None:
        self._set(experts, position.shape, torch.cat([position.flatten(), source, offsets, padded_offsets]))

    @classmethod
    def of_buffer(cls, experts: int, shape: torch.Size, buffer: torch.Tensor) -> "ExpertRouting":
        routing = cls.__new__(cls)
        routing._set(experts, shape, buffer)
        return routing

    def _set(self, experts: int, shape: torch.Size, buffer: torch.Tensor) -> None:
        self.experts = experts
        self.tokens, self.top_k = shape
        self.rows = self.tokens * self.top_k
        self.buffer = buffer

    @property
    def position(self) -> torch.Tensor:
        return self.buffer[: self.rows].view(self.tokens, self.top_k)

    @property
    def source(self) -> torch.Tensor:
        return self.buffer[self.rows : 2 * self.rows]

    @property
    def offsets(self) -> torch.Tensor:
        return self.buffer[2 * self.rows : 2 * self.rows + self.experts + 1]

    @property
    def padded_offsets(self) -> torch.Tensor:
        return self.buffer[2 * self.rows + self.experts + 1 :]

    def pointers(self) -> tuple[int, int, int, int]:
        """Device addresses of position, source, offsets and padded_offsets."""
        position = self.buffer.data_ptr()
        offsets = position + 8 * self.rows
        return position, position + 4 * self.rows, offsets, offsets + 4 * (self.experts + 1)

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
    if not expert_ids.is_contiguous():
        expert_ids = expert_ids.contiguous()
    return ExpertRouting.of_buffer(experts, expert_ids.shape, hip_ops.expert_route_buffer(expert_ids, experts))


def differentiates(*tensors: torch.Tensor | None) -> bool:
    """Whether a call on these has to be recorded (or has to refuse a transform)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return torch._C._are_functorch_transforms_active() or forward_ad._current_level >= 0


def _check_device(routing: ExpertRouting, *tensors: torch.Tensor) -> None:
    hip_ops._require_gpu(routing.buffer, *tensors)


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, routing: ExpertRouting) -> torch.Tensor:
        ctx.routing = routing
        return _dispatch(x, routing)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad: torch.Tensor):
        routing = ctx.routing
        return hip_ops.expert_combine_at(grad.contiguous(), routing.pointers()[0], routing.tokens, routing.top_k), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, rows: torch.Tensor, weights: torch.Tensor, routing: ExpertRouting) -> torch.Tensor:
        ctx.routing = routing
        ctx.save_for_backward(rows, weights)
        return _combine(rows, weights, routing)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad: torch.Tensor):
        rows, weights = ctx.saved_tensors
        position, _, offsets, _ = ctx.routing.pointers()
        return (*hip_ops.expert_combine_backward_at(grad.contiguous(), rows, position, offsets, ctx.routing.experts, weights), None)


def _dispatch(x: torch.Tensor, routing: ExpertRouting) -> torch.Tensor:
    position, _, offsets, _ = routing.pointers()
    return hip_ops.expert_dispatch_at(x, position, offsets, routing.experts, routing.top_k)


def _combine(rows: torch.Tensor, weights: torch.Tensor, routing: ExpertRouting) -> torch.Tensor:
    return hip_ops.expert_combine_at(rows, routing.pointers()[0], routing.tokens, routing.top_k, weights)


def dispatch_tokens(x: torch.Tensor, routing: ExpertRouting) -> torch.Tensor:
    """The tokens' rows [tokens, width] (bf16, fp16 or fp32) gathered into sorted
    rows [tokens * top_k, width], differentiable: a token's gradient is the sum of
    its rows' gradients, in fp32 in the order of its choices."""
    if x.ndim != 2 or x.shape[0] != routing.tokens:
        raise ValueError(f"x must be [{routing.tokens}, width], got {tuple(x.shape)}")
    _check_device(routing, x)
    x = x.contiguous()
    return _Dispatch.apply(x, routing) if differentiates(x) else _dispatch(x, routing)


def combine_tokens(rows: torch.Tensor, routing: ExpertRouting, weights: torch.Tensor) -> torch.Tensor:
    """``out[t] = sum_j weights[t, j] * rows[position[t, j]]`` for sorted rows
    [tokens * top_k, width], differentiable in both; fp32 sums in the order of j,
    rounded once.  A token none of whose experts are here gets zeros."""
    if rows.ndim != 2 or rows.shape[0] != routing.rows:
        raise ValueError(f"rows must be [{routing.rows}, width], got {tuple(rows.shape)}")
    if tuple(weights.shape) != (routing.tokens, routing.top_k):
        raise ValueError(f"weights must be {(routing.tokens, routing.top_k)}, got {tuple(weights.shape)}")
    _check_device(routing, rows, weights)
    rows, weights = rows.contiguous(), weights.contiguous()
    return _Combine.apply(rows, weights, routing) if differentiates(rows, weights) else _combine(rows, weights, routing)


__all__ = ["ExpertRouting", "combine_tokens", "dispatch_tokens", "route_tokens"]
