"""AdamW's 8-bit states as they are defined, on the CPU, and one step in 64 bits."""

import math

import torch

BLOCK = 128
FIRST, SECOND = 127, 255  # the largest code of each moment


def dither(count, t, codes):
    """The 32-bit fractions that rounding goes by at step ``t``."""
    z = (torch.arange(count) * 0x9E3779B9 + t * 0x6A09E667) % 2**32
    z = (z ^ (z >> 16)) * 0xBB67AE85 % 2**32
    z = z ^ (z >> 15)
    return ((z if codes == FIRST else z >> 16) & 0xFFFF) << 16


def encode(x, t, codes):
    """uint8 codes and fp32 scales of a flat fp32 tensor at step ``t``."""
    n = x.numel()
    blocks = torch.zeros(-(-n // BLOCK) * BLOCK)
    blocks[:n] = x
    scale = blocks.view(-1, BLOCK).abs().amax(dim=1).clamp(min=2.0**-100)
    inverse = torch.ones_like(scale) / scale
    size = (blocks.abs().view(-1, BLOCK) * inverse[:, None]).clamp(max=1.0).view(-1)
    u = dither(blocks.numel(), t, codes)
    code = ((size.view(torch.int32).long() + (u >> 12)) >> 20) - (1016 - codes)
    if codes == FIRST:
        smallest = 1.25 * 2.0**-16
        few = (size * torch.tensor(1 / smallest) > (u >> 8).float() * 2.0**-24).long()
        code = torch.where(size < smallest, few, code) + torch.where(blocks < 0, 128, 0)
    else:
        code = torch.where(size > 0, code.clamp(min=1), 0)
    return (code[:n] & 255).to(torch.uint8), scale


def decode(code, scale, codes):
    """fp32 values of flat codes."""
    n, code = code.numel(), code.int()
    size = code & 127 if codes == FIRST else code
    value = torch.where(size > 0, (size + 1016 - codes) << 20, 0).view(torch.float32)
    if codes == FIRST:
        value = torch.where(code > 127, -value, value)
    return value * scale.repeat_interleave(BLOCK)[:n]


def step64(p, g, m, v, t, *, lr, betas, eps, weight_decay, clip=1.0):
    """The step in 64 bits: new p, m, v."""
    b1, b2 = betas
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * clip
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    p = p * (1 - lr * weight_decay) - lr / (1 - b1**t) * m / (torch.sqrt(v) / math.sqrt(1 - b2**t) + eps)
    return p, m, v
