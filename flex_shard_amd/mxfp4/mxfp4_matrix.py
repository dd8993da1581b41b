"""Matrices of microscaled 4-bit floats: E2M1 elements (magnitudes 0, 0.5, 1,
1.5, 2, 3, 4, 6), 32 consecutive ones of a row under one power of two.

A run's scale is the power of two of its largest magnitude, less 2, as a byte
(its exponent + 127; 255 for a run with an infinity or a NaN, all of which then
stands for NaN).  Elements round to nearest, ties to the even code, and stop at 6.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import hip_ops
from ..hip_ops import MxFp4Matrix


def as_rows(x: torch.Tensor) -> torch.Tensor:
    """A matrix with contiguous, separate rows, as the quantizers read it."""
    if x.ndim != 2:
        raise ValueError(f"expected a matrix, got {tuple(x.shape)}")
    if x.is_contiguous():
        return x
    (rows, cols), (along, across) = x.shape, x.stride()
    return x if (cols <= 1 or across == 1) and (rows <= 1 or along >= cols) else x.contiguous()


def mxfp4_quantize(x: torch.Tensor) -> MxFp4Matrix:
    """Quantize a bf16, fp16 or fp32 matrix in runs of 32 along its rows."""
    return hip_ops.mxfp4_quantize(as_rows(x))[0]


def mxfp4_quantize_transposed(x: torch.Tensor) -> MxFp4Matrix:
    """The transpose of ``x``, quantized in runs of 32 along the columns of ``x``:
    what a product over the rows of ``x`` reads."""
    return hip_ops.mxfp4_quantize(as_rows(x), rows=False, columns=True)[1]


def mxfp4_quantize_both(x: torch.Tensor) -> tuple[MxFp4Matrix, MxFp4Matrix]:
    """:func:`mxfp4_quantize` and :func:`mxfp4_quantize_transposed` from one read."""
    return hip_ops.mxfp4_quantize(as_rows(x), columns=True)[:2]


@dataclass(frozen=True)
class MxFp4Weight:
    """A linear layer's weight [out, in], or experts' weights [experts, out, in],
    quantized once; ``transposed`` (optional) is what an input gradient reads."""

    shape: tuple[int, ...]
    dtype: torch.dtype
    matrix: MxFp4Matrix
    transposed: MxFp4Matrix | None = None

    def __post_init__(self) -> None:
        if len(self.shape) not in (2, 3):
            raise ValueError(f"a weight is [out, in] or [experts, out, in], got {tuple(self.shape)}")
        *experts, rows, cols = self.shape
        count = experts[0] if experts else 1
        for form, want in ((self.matrix, (count * rows, cols)), (self.transposed, (count * cols, rows))):
            if form is not None and (form.rows, form.cols) != want:
                raise ValueError(f"a weight {tuple(self.shape)} has a form {want}, got {(form.rows, form.cols)}")


def quantize_mxfp4_weight(weight: torch.Tensor, *, transposed: bool = False) -> MxFp4Weight:
    """Quantize a weight that stays as it is: serving, or a frozen layer
    (``transposed``: gradients pass through it to its input)."""
    if weight.ndim not in (2, 3):
        raise ValueError(f"expected a weight [out, in] or [experts, out, in], got {tuple(weight.shape)}")
    source = as_rows(weight) if weight.ndim == 2 else weight.contiguous()
    rows, columns, _ = hip_ops.mxfp4_quantize(source.detach(), columns=transposed)
    return MxFp4Weight(tuple(weight.shape), weight.dtype, rows, columns)


__all__ = [
    "MxFp4Matrix", "MxFp4Weight", "mxfp4_quantize", "mxfp4_quantize_both", "mxfp4_quantize_transposed", "quantize_mxfp4_weight",
]
