"""An activation that is already quantized when a linear reads it."""

from __future__ import annotations

from typing import Any, Callable, Sequence

import torch

from .. import hip_ops


class Fp8Activation:
    """Rows of E4M3 bytes with a scale for every run of 128 columns, as the FP8
    linear's quantizer writes them: ``q`` float8_e4m3fn [rows, cols rounded up to
    128], ``scales`` fp32 [that / 128, rows], for an activation of ``shape`` [..., cols].

    ``FlexShardFloat8BlockwiseLinear`` and ``prequantized_linear`` take one in place of
    an activation.  ``carrier`` stands for it in autograd: a bf16 tensor of that
    shape without values of its own, through which the linears' gradients reach what
    made the activation, unrounded by the quantizer (straight through).  (Reentrant
    checkpointing sees tensors alone: make and read one inside the same region, or hand on ``dequantize()``.)"""

    __slots__ = ("q", "scales", "shape", "carrier", "_make_runs", "_sources", "_runs", "_captured")

    def __init__(
        self, q: torch.Tensor, scales: torch.Tensor, carrier: torch.Tensor,
        make_token_runs: Callable[[], tuple[torch.Tensor, torch.Tensor]], sources: Sequence[torch.Tensor] = (),
    ) -> None:
        self.q = q
        self.scales = scales
        self.shape = carrier.shape
        self.carrier = carrier
        self._make_runs = make_token_runs
        self._sources = sources  # (what that reads)
        self._runs: tuple | None = None
        self._captured = q.is_cuda and torch.cuda.is_current_stream_capturing()

    @property
    def ndim(self) -> int:
        return len(self.shape)

    @property
    def device(self) -> torch.device:
        return self.q.device

    def token_runs(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The activation in runs of 128 tokens, transposed, with its scales: what a
        weight gradient contracts over.  Made when the first linear asks for it, for
        all that do so on the same stream (but anew for a capture that the activation
        is not part of: a graph's memory holds nothing before its first replay)."""
        if torch.cuda.is_current_stream_capturing() != self._captured:
            return self._make_runs()
        stream = hip_ops.stream_ptr(self.q.device)
        if self._runs is None or self._runs[0] != stream:
            self._runs = (stream, self._make_runs())
        return self._runs[1]

    def record_stream(self, stream: torch.cuda.Stream) -> None:
        """As for a tensor: what work on ``stream`` reads is not reused before that work is done."""
        for t in (self.q, self.scales, *self._sources):
            t.record_stream(stream)

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values, differentiable straight through the quantizer."""
        if torch.is_grad_enabled() and self.carrier.requires_grad:
            return _Dequantize.apply(self.carrier, self, dtype)
        return self._values(dtype)

    def _values(self, dtype: torch.dtype) -> torch.Tensor:
        return hip_ops.act_dequant_1x128(self.q, self.scales, self.shape[-1], dtype, self.shape)

    def __repr__(self) -> str:
        return f"Fp8Activation(shape={tuple(self.shape)})"


class _Dequantize(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, carrier: torch.Tensor, activation: Fp8Activation, dtype: torch.dtype) -> torch.Tensor:
        return activation._values(dtype)

    @staticmethod
    def backward(ctx: Any, grad: torch.Tensor):  # (linear in the gradient: differentiable again)
        return grad if grad.dtype is torch.bfloat16 else grad.to(torch.bfloat16), None, None


__all__ = ["Fp8Activation"]
