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

from .. import _native, hip_ops


class ExpertRouting:
    """The choices [tokens, top_k] of a router in stable order by expert.  There
    are tokens * top_k sorted rows; rows from ``offsets[-1]`` on belong to choices
    of no expert here, hold nothing, and are zero wherever they are written.

    ``position`` [tokens, top_k]: the sorted row of each choice, -1 for no expert
    here.  ``offsets`` [experts + 1]: expert ``e`` has rows ``offsets[e]`` to
    ``offsets[e + 1]``.  ``source`` [tokens * top_k]: the choice ``t * top_k + j`` of
    each sorted row, -1 behind the last.  ``padded_offsets`` [experts + 1]: the
    segments, each rounded up to 256 rows (a product over an expert's rows).  All
    int32, behind one another in one buffer.

    :func:`route_tokens` makes them.  Kernels index by what the tables hold, so
    tables of another origin are checked before the first use of a routing
    (:meth:`check`), which waits for the GPU once."""

    __slots__ = ("experts", "tokens", "top_k", "rows", "buffer", "_sizes", "_checked")

    def __init__(
        self, experts: int, position: torch.Tensor, offsets: torch.Tensor, source: torch.Tensor, padded_offsets: torch.Tensor
    ) -> None:
        tables = (position.flatten(), source.flatten(), offsets.flatten(), padded_offsets.flatten())
        self._set(experts, position.shape, torch.cat(tables), tuple(t.numel() for t in tables))

    @classmethod
    def of_buffer(cls, experts: int, shape: torch.Size, buffer: torch.Tensor) -> "ExpertRouting":
        routing = cls.__new__(cls)
        routing._set(experts, shape, buffer, None)
        return routing

    def _set(self, experts: int, shape: torch.Size, buffer: torch.Tensor, sizes: tuple[int, ...] | None) -> None:
        self.experts = experts
        self.tokens, self.top_k = shape
        self.rows = self.tokens * self.top_k
        self.buffer = buffer
        self._sizes = sizes
        self._checked = False

    def check(self) -> None:
        """Raise ``ValueError`` unless the tables are an order of the choices by
        expert as described above.  Nothing to do for those of :func:`route_tokens`."""
        if not self._checked:
            self._check_tables()
            self._checked = True

    def _check_tables(self) -> None:
        experts, rows, buffer = self.experts, self.rows, self.buffer
        if not 1 <= experts <= _native.MAX_EXPERTS or self.top_k < 1:
            raise ValueError(f"a routing has 1 to {_native.MAX_EXPERTS} experts and at least one choice per token, got {experts}, {self.top_k}")
        sizes = (rows, rows, experts + 1, experts + 1)
        if buffer.dtype != torch.int32:
            raise ValueError(f"a routing's tables are int32, got {buffer.dtype}")
        if buffer.ndim != 1 or not buffer.is_contiguous() or buffer.numel() != sum(sizes) or self._sizes not in (None, sizes):
            raise ValueError(
                f"position, source, offsets and padded_offsets must have {sizes} elements, got {self._sizes or tuple(buffer.shape)}"
            )
        position, source, offsets, padded = (t.long() for t in buffer.split(sizes))
        row = torch.arange(rows, device=buffer.device)
        used = offsets[-1]
        here = row < used
        lengths = offsets.diff()
        right = (
            (offsets[0] == 0) & (lengths >= 0).all() & (used <= rows)
            # as many choices with a row as there are rows, and each row that of its choice: one to one
            & ((position >= -1) & (position < rows)).all() & ((position >= 0).sum() == used)
            & torch.where(here, (source >= 0) & (source < rows), source == -1).all()
            & ((position[source.clamp(0, max(rows - 1, 0))] == row) | ~here).all()
            & (padded[0] == 0) & (padded.diff() == (lengths + 255) // 256 * 256).all()
        )
        if not bool(right):
            raise ValueError("position, offsets, source and padded_offsets are not one order of the choices by expert")

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
        self.check()
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
    routing = ExpertRouting.of_buffer(experts, expert_ids.shape, hip_ops.expert_route_buffer(expert_ids, experts))
    routing._checked = True
    return routing


def differentiates(*tensors: torch.Tensor | None) -> bool:
    """Whether a call on these has to be recorded (or has to refuse a transform)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return torch._C._are_functorch_transforms_active() or forward_ad._current_level >= 0


def check_routing(routing: ExpertRouting, *tensors: torch.Tensor) -> None:
    """The routing's tables and the tensors of a call are on one GPU, and the tables in order."""
    hip_ops._require_gpu(routing.buffer, *tensors)
    routing.check()


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
    check_routing(routing, x)
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
    check_routing(routing, rows, weights)
    rows, weights = rows.contiguous(), weights.contiguous()
    return _Combine.apply(rows, weights, routing) if differentiates(rows, weights) else _combine(rows, weights, routing)


__all__ = ["ExpertRouting", "combine_tokens", "dispatch_tokens", "route_tokens"]
