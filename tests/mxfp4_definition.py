"""Microscaled 4-bit floats by their definition, in float64 on the CPU: what the
GPU tests compare with."""

import torch

VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize(x: torch.Tensor):
    """Codes (sign * 8 + magnitude, [rows, cols padded to 256]) and scale bytes
    ([rows, cols padded / 32]) of a matrix, in runs of 32 along its rows."""
    rows, cols = x.shape
    padded = -(-cols // 256) * 256
    full = torch.zeros(rows, padded, dtype=torch.float64)
    full[:, :cols] = x.double().cpu()
    runs = full.view(rows, padded // 32, 32)
    finite = torch.isfinite(runs).all(dim=-1)
    size = torch.where(torch.isfinite(runs), runs.abs(), 0.0)
    largest = size.amax(dim=-1)
    _, exponent = torch.frexp(largest)  # largest = m * 2**exponent, m in [0.5, 1)
    byte = torch.where(largest > 0, exponent - 1 - 2 + 127, 0).clamp(min=0)
    scaled = size / torch.exp2(byte.double() - 127)[..., None]
    distance = (scaled[..., None] - VALUES).abs()
    best = distance.min(dim=-1, keepdim=True).values
    tied = distance == best  # one code, or two neighbours of which one is even
    code = torch.arange(8)
    magnitude = torch.where(tied & (code % 2 == 0), code, -1).amax(dim=-1)
    magnitude = torch.where(magnitude < 0, torch.where(tied, code, -1).amax(dim=-1), magnitude)
    codes = magnitude + 8 * torch.signbit(runs).long()
    return codes.view(rows, padded), torch.where(finite, byte, 255)


def values(codes: torch.Tensor, byte: torch.Tensor, cols: int) -> torch.Tensor:
    """What codes and scale bytes stand for."""
    scale = torch.where(byte == 255, torch.nan, torch.exp2(byte.double() - 127)).repeat_interleave(32, dim=1)
    sign = torch.where(codes >= 8, -1.0, 1.0).double()
    return (sign * VALUES[codes % 8] * scale)[:, :cols]


def through(x: torch.Tensor) -> torch.Tensor:
    return values(*quantize(x), x.shape[1])


def unpack(data: torch.Tensor, scales: torch.Tensor):
    """Codes and bytes out of a matrix as it lies in memory."""
    data, scales = data.cpu().long(), scales.cpu().long()
    codes = torch.stack([data & 15, data >> 4], dim=-1).flatten(1)
    return codes, scales.permute(1, 0, 2).flatten(1)


#: unit roundoff of the output types
ROUNDING = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def assert_product(got: torch.Tensor, a: torch.Tensor, b: torch.Tensor, extra: torch.Tensor | None = None, terms: int = 0) -> None:
    """``got`` is a @ b.T (+ extra) of float64 values within what k fp32 additions,
    each off by at most 2**-23 of the sum of magnitudes, and one rounding allow."""
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    if extra is not None:
        want, size = want + extra, size + extra.abs()
    got64 = got.double().cpu()
    assert got64.shape == want.shape
    bound = (a.shape[1] + terms) * 2.0**-23 * size + ROUNDING[got.dtype] * want.abs() + 2.0**-133
    if got.dtype == torch.float16:
        bound = bound + 2.0**-25  # half a subnormal step
    worst = ((got64 - want).abs() - bound).max().item() if want.numel() else -1.0
    assert worst <= 0.0, worst
