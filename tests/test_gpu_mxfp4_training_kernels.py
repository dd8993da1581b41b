"""The kernels that training steps of usual sizes take: large tiles in every type, over the rows of experts of which some
have none, and in all three products of an experts' layer."""

import pytest
import torch
from mxfp4_definition import ROUNDING

from flex_shard_amd import _native, hip_ops
from flex_shard_amd.experts import route_tokens
from flex_shard_amd.mxfp4 import mxfp4_expert_linear, mxfp4_quantize

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _values(t):
    """What the rows of ``t`` stand for in 4 bits, in 64 bits (the quantizers have their own tests, bit for bit)."""
    return mxfp4_quantize(t.contiguous()).dequantize(torch.float32).double()


def _assert_close(got, a, b, terms=0):
    """``got`` is a @ b.T within what one fp32 addition per column, each off by at most 2**-23 of the sum of magnitudes,
    and one rounding allow."""
    want, size = torch.mm(a, b.t()), torch.mm(a.abs(), b.abs().t())
    bound = (a.shape[1] + terms) * 2.0**-23 * size + ROUNDING[got.dtype] * want.abs()
    if got.dtype == torch.float16:
        bound += 2.0**-25
    assert ((got.double() - want).abs() <= bound).all()


LENGTHS = [0, 1, 255, 256, 0, 257, 512, 1300, 0, 0, 513, 40, 770, 1024, 0, 256]  # none to six steps of 256


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(
    "tiles,m,n,lengths",
    [
        ("256", 1030, 1290, LENGTHS),  # 480 tiles: a workgroup takes one of no steps, one of some, and ends inside them
        ("256", 1280, 1536, LENGTHS),  # whole tiles
        ("256", 777, 1500, LENGTHS + LENGTHS[::-1]),
        ("256", 1030, 1290, [0] * 15 + [300]),
        ("256", 1030, 1290, [2000] + [0] * 15),
        ("256", 520, 2060, [0, 600, 0, 0, 1, 0, 256, 0]),
        ("128 deep", 300, 700, LENGTHS[:12]),
        ("128", 1030, 1290, LENGTHS[:12]),
        ("64", 300, 700, LENGTHS[:8]),
    ],
)
def test_over_rows(device, tiles, m, n, lengths, dtype):
    experts, rows = len(lengths), sum(lengths)
    padded = [-(-count // 256) * 256 for count in lengths]
    # (as many as a routing sets aside: more than the segments take)
    padded_rows = (rows + 255 * experts) // 256 * 256
    assert hip_ops.mxfp4_gemm_tiles(m, n, padded_rows, mode=_native.MXFP4_OVER_ROWS, experts=experts) == tiles
    offsets = torch.tensor([0] + lengths).cumsum(0).to(device, torch.int32)
    padded_offsets = torch.tensor([0] + padded).cumsum(0).to(device, torch.int32)
    gen = torch.Generator(device=device).manual_seed(m + rows)
    g, x = (torch.randn(rows, width, generator=gen, device=device).to(dtype) for width in (m, n))
    a, b = (hip_ops.mxfp4_quantize_segments(t, offsets, padded_offsets, padded_rows, choices=rows)[1] for t in (g, x))
    got = hip_ops.mxfp4_gemm(a, b, dtype, mode=_native.MXFP4_OVER_ROWS, offsets=padded_offsets)
    assert got.shape == (experts, m, n) and got.dtype == dtype
    at = 0
    for e, count in enumerate(lengths):
        if count:
            part = slice(at, at + count)
            _assert_close(got[e], _values(g[part].t()), _values(x[part].t()))
        else:
            assert not got[e].any()
        at += count
    assert torch.equal(got, hip_ops.mxfp4_gemm(a, b, dtype, mode=_native.MXFP4_OVER_ROWS, offsets=padded_offsets))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sorted_rows", [False, True])
@pytest.mark.parametrize("out_dim,in_dim", [(520, 2060), (768, 2048)])
def test_all_three_products_of_an_experts_layer(device, out_dim, in_dim, sorted_rows, dtype):
    tokens, top_k, experts = 5000, 4, 8
    rows = tokens * top_k
    padded_rows = (rows + 255 * experts) // 256 * 256
    for sizes, mode in (((rows, out_dim, in_dim), _native.MXFP4_ROWS), ((rows, in_dim, out_dim), _native.MXFP4_ROWS),
                        ((out_dim, in_dim, padded_rows), _native.MXFP4_OVER_ROWS)):
        assert hip_ops.mxfp4_gemm_tiles(*sizes, mode=mode, experts=experts) == "256"
    gen = torch.Generator(device=device).manual_seed(out_dim)
    ids = torch.randint(0, experts, (tokens, top_k), generator=gen, device=device)
    ids = torch.where((ids == 2) | (ids == 5), -1, ids)  # two experts without rows, and rows of no expert
    ids[(ids == 3).cumsum(1).cumsum(0) > 1] = 6  # one with very few
    routing = route_tokens(ids, experts)
    x = torch.randn(rows if sorted_rows else tokens, in_dim, generator=gen, device=device).to(dtype).requires_grad_()
    w = (torch.randn(experts, out_dim, in_dim, generator=gen, device=device) * 0.05).to(dtype).requires_grad_()
    g = torch.randn(rows, out_dim, generator=gen, device=device).to(dtype)
    y = mxfp4_expert_linear(x, w, routing, sorted_rows=sorted_rows)
    gx, gw = torch.autograd.grad(y, (x, w), g)
    offsets, source = routing.offsets.tolist(), routing.source.long()
    assert offsets[3] == offsets[2] and offsets[6] == offsets[5] and offsets[-1] < rows
    x, w, y = x.detach(), w.detach(), y.detach()
    want = torch.zeros(x.shape, dtype=torch.float64, device=device)
    size = torch.zeros_like(want)
    for e in range(experts):
        part = slice(offsets[e], offsets[e + 1])
        if part.start == part.stop:
            assert not gw[e].any()
            continue
        of = torch.arange(part.start, part.stop, device=device) if sorted_rows else source[part] // top_k
        _assert_close(y[part], _values(x[of]), _values(w[e]))
        _assert_close(gw[e], _values(g[part].t()), _values(x[of].t()))
        a, b = _values(g[part]), _values(w[e].t())
        want.index_add_(0, of, torch.mm(a, b.t()))
        size.index_add_(0, of, torch.mm(a.abs(), b.abs().t()))
    assert not y[offsets[-1] :].any()
    bound = (out_dim + top_k) * 2.0**-23 * size + ROUNDING[dtype] * want.abs() + (2.0**-25 if dtype == torch.float16 else 0.0)
    assert ((gx.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("m,n,k", [(8001, 4091, 1030), (8190, 4088, 520), (4096, 8192, 1792), (7950, 4096, 200)])
def test_fp16_of_large_dense_tiles(device, m, n, k):
    assert hip_ops.mxfp4_gemm_tiles(m, n, k) == "256"
    gen = torch.Generator(device=device).manual_seed(m)
    a, b = (mxfp4_quantize(torch.randn(rows, k, generator=gen, device=device)) for rows in (m, n))
    bias = torch.randn(n, generator=gen, device=device)
    # the same sums, whose fp32 results have a test of their own, rounded once more
    assert torch.equal(hip_ops.mxfp4_gemm(a, b, torch.float16, bias=bias), hip_ops.mxfp4_gemm(a, b, torch.float32, bias=bias).half())
    assert torch.equal(hip_ops.mxfp4_gemm(a, b, torch.float16), hip_ops.mxfp4_gemm(a, b, torch.float32).half())


@pytest.mark.parametrize("tiles,tokens,out_dim", [("64", 60, 40), ("128", 40000, 264)])
def test_as_many_experts_as_a_tile_has_a_table_for(device, tiles, tokens, out_dim):
    experts, top_k, in_dim = _native.MAX_EXPERTS, 2, 64
    assert hip_ops.mxfp4_gemm_tiles(tokens * top_k, out_dim, in_dim, mode=_native.MXFP4_ROWS, experts=experts) == tiles
    gen = torch.Generator(device=device).manual_seed(tokens)
    ids = torch.randint(-1, experts, (tokens, top_k), generator=gen, device=device)
    ids[0] = torch.tensor([0, experts - 1], device=device)
    routing = route_tokens(ids, experts)
    x, w = torch.randn(tokens, in_dim, generator=gen, device=device), torch.randn(experts, out_dim, in_dim, generator=gen, device=device)
    with torch.no_grad():
        y = mxfp4_expert_linear(x, w, routing)
    used = int(routing.offsets[-1])
    source = routing.source[:used].long()
    expert = ids.flatten()[source]
    x64, w64 = _values(x), _values(w.view(-1, in_dim)).view(w.shape)
    for first in range(0, used, 1000):
        part = slice(first, min(first + 1000, used))
        a, b = x64[source[part] // top_k], w64[expert[part]]
        want, size = (b * a[:, None]).sum(-1), (b * a[:, None]).abs().sum(-1)
        assert ((y[part].double() - want).abs() <= in_dim * 2.0**-23 * size + ROUNDING[y.dtype] * want.abs()).all()
    assert not y[used:].any()
