"""The input gradient of an experts' layer on unsorted tokens: the choices' parts are added up in fp32 and rounded once."""

import pytest
import torch
from mxfp4_definition import ROUNDING, through

from flex_shard_amd import _native, hip_ops
from flex_shard_amd.experts import route_tokens
from flex_shard_amd.mxfp4 import mxfp4_expert_linear, mxfp4_quantize

pytestmark = pytest.mark.gpu


def _gradient(x, w, ids, g):
    leaf = x.requires_grad_()
    y = mxfp4_expert_linear(leaf, w, route_tokens(ids, w.shape[0]))
    return torch.autograd.grad(y, leaf, g)[0]


@pytest.mark.parametrize("width", [32, 33, 40])
def test_fp16_parts_beyond_its_range_whose_sum_is_not(device, width):
    # A part is 4096 * 24 * 32, 48 times the largest fp16; the other expert's takes all of it away but 4096 * 8.
    # All values are 4-bit elements times a power of two, so that nothing is rounded anywhere.
    w = torch.full((2, 32, width), 24.0, dtype=torch.float16, device=device)
    w[1] = -24.0
    w[1, 5] = -16.0
    ids = torch.tensor([[0, 1], [1, 0], [0, 1]], device=device)
    g = torch.full((6, 32), 4096.0, dtype=torch.float16, device=device)
    got = _gradient(torch.ones(3, width, dtype=torch.float16, device=device), w, ids, g)
    assert got.dtype == torch.float16 and torch.equal(got, torch.full_like(got, 4096.0 * 8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,top_k,experts,out_dim,in_dim", [(1, 8, 16, 96, 320), (33, 3, 7, 65, 257), (50, 1, 4, 64, 96), (20, 9, 12, 130, 72)])
def test_one_rounding(device, tokens, top_k, experts, out_dim, in_dim, dtype):
    gen = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-1, experts, (tokens, top_k), generator=gen)
    x, w = torch.randn(tokens, in_dim, generator=gen).to(dtype), (torch.randn(experts, out_dim, in_dim, generator=gen) * 0.05).to(dtype)
    g = torch.randn(tokens * top_k, out_dim, generator=gen).to(dtype)
    got = _gradient(x.to(device), w.to(device), ids.to(device), g.to(device))
    want, size = torch.zeros(tokens, in_dim, dtype=torch.float64), torch.zeros(tokens, in_dim, dtype=torch.float64)
    flat, at = ids.flatten(), 0
    for e in range(experts):
        choices = (flat == e).nonzero().flatten()
        a, b = through(g[at : at + len(choices)]), through(w[e].t())
        want.index_add_(0, choices // top_k, a @ b.t())
        size.index_add_(0, choices // top_k, a.abs() @ b.abs().t())
        at += len(choices)
    # out_dim and top_k fp32 additions, each off by at most 2**-23 of the sum of magnitudes, and one rounding
    bound = (out_dim + top_k) * 2.0**-23 * size + ROUNDING[dtype] * want.abs() + (2.0**-25 if dtype == torch.float16 else 2.0**-133)
    assert ((got.double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_rounding_of_large_tiles(device, dtype):
    tokens, top_k, experts, out_dim, in_dim = 2500, 4, 6, 520, 1300
    tiles = hip_ops.mxfp4_gemm_tiles(tokens * top_k, in_dim, out_dim, mode=_native.MXFP4_ROWS, experts=experts)
    assert tiles == "256"
    gen = torch.Generator(device=device).manual_seed(5)
    ids = torch.randint(-1, experts, (tokens, top_k), generator=gen, device=device)
    x = torch.randn(tokens, in_dim, generator=gen, device=device).to(dtype)
    w = (torch.randn(experts, out_dim, in_dim, generator=gen, device=device) * 0.05).to(dtype)
    g = torch.randn(tokens * top_k, out_dim, generator=gen, device=device).to(dtype)
    got = _gradient(x, w, ids, g)
    routing = route_tokens(ids, experts)
    offsets, source = routing.offsets.tolist(), routing.source.long()
    want = torch.zeros(tokens, in_dim, dtype=torch.float64, device=device)
    size = torch.zeros_like(want)
    for e in range(experts):
        part = slice(offsets[e], offsets[e + 1])
        a = mxfp4_quantize(g[part]).dequantize(torch.float32).double()
        b = mxfp4_quantize(w[e].t()).dequantize(torch.float32).double()
        want.index_add_(0, source[part] // top_k, torch.mm(a, b.t()))
        size.index_add_(0, source[part] // top_k, torch.mm(a.abs(), b.abs().t()))
    bound = (out_dim + top_k) * 2.0**-23 * size + ROUNDING[dtype] * want.abs() + (2.0**-25 if dtype == torch.float16 else 2.0**-133)
    assert ((got.double() - want).abs() <= bound).all()
