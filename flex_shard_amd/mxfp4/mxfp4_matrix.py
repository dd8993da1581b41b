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


@dataclass(frozen=True)
class MxFp4Matrix:
    """A quantized matrix.  ``data`` is uint8 [rows, P / 2], P = ``cols`` rounded up
    to 256 (the lower column in a byte's low half, the pad zero); ``scales`` uint8
    [P / 256, rows, 8], the bytes of a row's 256 columns next to one another."""

    data: torch.Tensor
    scales: torch.Tensor
    cols: int

    @property
    def rows(self) -> int:
        return self.data.shape[0]

    @property
    def pair(self) -> tuple[torch.Tensor, torch.Tensor]:
        return self.data, self.scales

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values [rows, cols] in bf16, fp16 or fp32."""
        return hip_ops.mxfp4_dequantize(self.data, self.scales, self.cols, dtype)


def as_rows(x: torch.Tensor) -> torch.Tensor:
    """A matrix with contiguous, separate rows, as the quantizers read it."""
    if x.ndim != 2:
        raise ValueError(f"expected a matrix, got {tuple(x.shape)}")
    if (x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        return x.contiguous()
    return x


def mxfp4_quantize(x: torch.Tensor) -> MxFp4Matrix:
    """Quantize a bf16, fp16 or fp32 matrix in runs of 32 along its rows."""
    x = as_rows(x)
    rows, _, _ = hip_ops.mxfp4_quantize(x)
    return MxFp4Matrix(*rows, x.shape[1])


def mxfp4_quantize_transposed(x: torch.Tensor) -> MxFp4Matrix:
    """The transpose of ``x``, quantized in runs of 32 along the columns of ``x``:
    what a product over the rows of ``x`` reads."""
    x = as_rows(x)
    _, columns, _ = hip_ops.mxfp4_quantize(x, rows=False, columns=True)
    return MxFp4Matrix(*columns, x.shape[0])


def mxfp4_quantize_both(x: torch.Tensor) -> tuple[MxFp4Matrix, MxFp4Matrix]:
    """:func:`mxfp4_quantize` and :func:`mxfp4_quantize_transposed` from one read."""
    x = as_rows(x)
    rows, columns, _ = hip_ops.mxfp4_quantize(x, columns=True)
    return MxFp4Matrix(*rows, x.shape[1]), MxFp4Matrix(*columns, x.shape[0])


@dataclass(frozen=True)
class MxFp4Weight:
    """A linear layer's weight [out, in], or experts' weights [experts, out, in],
    quantized once; ``transposed`` (optional) is what an input gradient reads."""

    shape: tuple[int, ...]
    dtype: torch.dtype
    matrix: MxFp4Matrix
    transposed: MxFp4Matrix | None = None


def quantize_mxfp4_weight(weight: torch.Tensor, *, transposed: bool = False) -> MxFp4Weight:
    """Quantize a weight that stays as it is: serving, or a frozen layer
    (``transposed``: gradients pass through it to its input)."""
    if weight.ndim not in (2, 3):
        raise ValueError(f"expected a weight [out, in] or [experts, out, in], got {tuple(weight.shape)}")
    with torch.no_grad():
        source = as_rows(weight) if weight.ndim == 2 else weight.contiguous()
        rows, columns, _ = hip_ops.mxfp4_quantize(source, columns=transposed)
    out_dim, in_dim = weight.shape[-2:]
    return MxFp4Weight(
        tuple(weight.shape), weight.dtype, MxFp4Matrix(*rows, in_dim), MxFp4Matrix(*columns, out_dim) if transposed else None
    )


__all__ = [
    "MxFp4Matrix", "MxFp4Weight", "mxfp4_quantize", "mxfp4_quantize_both", "mxfp4_quantize_transposed", "quantize_mxfp4_weight",
]
