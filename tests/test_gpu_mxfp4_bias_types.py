"""A bias of another type than the activation is added to the fp32 sums as it is: one rounding, that of the result."""

import pytest
import torch
from mxfp4_definition import assert_product, through

from flex_shard_amd import hip_ops
from flex_shard_amd.mxfp4 import mxfp4_linear, quantize_mxfp4_weight

pytestmark = pytest.mark.gpu

HALVES = [torch.bfloat16, torch.float16]


# a size for every kernel of the dense product
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize(
    "tiles,m,n,k",
    [("few rows", 1, 130, 96), ("few rows", 4, 1001, 300), ("few rows", 16, 1001, 5000), ("64", 50, 3001, 1100), ("128", 1000, 5123, 600),
     ("128 deep", 2035, 2041, 700), ("256", 8001, 4091, 1030)],
)
def test_low_bits_of_an_fp32_bias_survive(device, tiles, m, n, k, dtype):
    assert hip_ops.mxfp4_gemm_tiles(m, n, k) == tiles
    x, w = torch.zeros(m, k, dtype=dtype, device=device), torch.zeros(n, k, dtype=dtype, device=device)
    x[:, 7], w[:, 7] = 1.0, -1.0
    small = (torch.arange(n, device=device) % 200) * 2.0**-14
    want = small.to(dtype).expand(m, n)  # -1 + (1 + small), eight bits of it
    frozen = quantize_mxfp4_weight(w)
    bias = 1.0 + small
    assert torch.equal(mxfp4_linear(x, frozen, bias), want)
    leaves = [w.requires_grad_(), bias.requires_grad_()]  # the training call quantizes ahead of the product
    y = mxfp4_linear(x, *leaves)
    assert y.dtype == dtype and torch.equal(y, want)
    gw, gb = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert gw.dtype == dtype and gb.dtype == torch.float32 and torch.equal(gb, torch.full_like(gb, m))


def test_bf16_bias_beyond_fp16(device):
    x, w = torch.zeros(3, 64, dtype=torch.float16, device=device), torch.zeros(40, 64, dtype=torch.float16, device=device)
    x[:, 1], w[:, 1] = 256.0, -512.0
    bias = torch.full((40,), 131072.0 + 1024.0, dtype=torch.bfloat16, device=device)  # an infinity in fp16
    assert torch.equal(mxfp4_linear(x, w, bias), torch.full((3, 40), 1024.0, dtype=torch.float16, device=device))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("bias_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [1, 4, 9, 200])
def test_against_the_unrounded_sum(device, tokens, bias_dtype, dtype):
    gen = torch.Generator().manual_seed(tokens)
    x, w = torch.randn(tokens, 96, generator=gen).to(dtype), (torch.randn(70, 96, generator=gen) * 0.05).to(dtype)
    bias = torch.randn(70, generator=gen).to(bias_dtype)
    got = mxfp4_linear(x.to(device), w.to(device), bias.to(device))
    assert got.dtype == dtype
    assert_product(got, through(x), through(w), bias.double())
    strided = torch.randn(70, 2, generator=gen).to(bias_dtype)
    got = mxfp4_linear(x.to(device), w.to(device), strided.to(device)[:, 1])
    assert_product(got, through(x), through(w), strided[:, 1].double())


def test_fp32_master_weight_and_bias(device):
    gen = torch.Generator().manual_seed(3)
    x, w, b = torch.randn(40, 96, generator=gen).bfloat16(), torch.randn(70, 96, generator=gen) * 0.05, torch.randn(70, generator=gen)
    g = (torch.randn(40, 70, generator=gen) * 0.01).bfloat16()
    leaves = [t.to(device).requires_grad_() for t in (x, w, b)]
    y = mxfp4_linear(*leaves)
    assert y.dtype == torch.bfloat16
    assert_product(y, through(x), through(w), b.double())
    gx, gw, gb = torch.autograd.grad(y, leaves, g.to(device))
    assert gx.dtype == torch.bfloat16 and gw.dtype == gb.dtype == torch.float32
    assert_product(gx, through(g), through(w.t()))
    assert_product(gw, through(g.t()), through(x.t()))
    assert ((gb.double().cpu() - g.double().sum(0)).abs() <= 41 * 2.0**-24 * g.double().abs().sum(0)).all()


@pytest.mark.parametrize("bias_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("needs_x", [False, True])
def test_bias_gradient_beside_a_frozen_weight(device, needs_x, bias_dtype):
    gen = torch.Generator().manual_seed(6)
    x, w = torch.randn(300, 96, generator=gen).bfloat16(), torch.randn(70, 96, generator=gen) * 0.05
    g, bias = torch.randn(300, 70, generator=gen).bfloat16(), torch.randn(70, generator=gen).to(bias_dtype)
    leaves = [bias.to(device).requires_grad_()] + ([x.to(device).requires_grad_()] if needs_x else [])
    y = mxfp4_linear(leaves[1] if needs_x else x.to(device), quantize_mxfp4_weight(w.to(device), transposed=needs_x), leaves[0])
    assert_product(y, through(x), through(w), bias.double())
    gb, *gx = torch.autograd.grad(y, leaves, g.to(device))
    size, want = g.double().abs().sum(0), g.double().sum(0)
    assert gb.dtype == bias_dtype
    assert ((gb.double().cpu() - want).abs() <= 300 * 2.0**-24 * size + (2.0**-8 if bias_dtype == torch.bfloat16 else 2.0**-24) * want.abs()).all()
    if needs_x:
        assert_product(gx[0], through(g), through(w.t()))
