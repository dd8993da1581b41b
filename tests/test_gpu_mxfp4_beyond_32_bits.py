"""Matrices and outputs whose elements and bytes pass 2^32: their far ends equal what small calls give."""

import pytest
import torch

from flex_shard_amd import hip_ops
from flex_shard_amd.experts import combine_tokens, dispatch_tokens, route_tokens
from flex_shard_amd.mxfp4 import mxfp4_expert_linear

pytestmark = pytest.mark.gpu


def test_quantize_both_ways_and_back(device):
    rows, cols = 70000, 65536
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=device)
    gen = torch.Generator(device=device).manual_seed(0)
    corner = torch.randn(300, 512, generator=gen, device=device).bfloat16()
    x[-300:, -512:] = corner
    row_form, column_form, _ = hip_ops.mxfp4_quantize(x, columns=True)
    # (a row's and a column's runs of 32 lie within the corner: 300 rows back from 70000 is no multiple of 32)
    want = hip_ops.mxfp4_quantize(corner)[0].dequantize()
    assert torch.equal(row_form.dequantize()[-300:, -512:], want)
    del row_form
    inner = corner[300 - rows % 32 - 256 :]
    want = hip_ops.mxfp4_quantize(inner, rows=False, columns=True)[1].dequantize()
    assert torch.equal(column_form.dequantize()[-512:, -inner.shape[0] :], want)


def test_product(device):
    m, n, k = 70000, 62000, 256
    gen = torch.Generator(device=device).manual_seed(1)
    a, b = (torch.randn(rows, k, generator=gen, device=device) for rows in (m, n))
    out = hip_ops.mxfp4_gemm(hip_ops.mxfp4_quantize(a)[0], hip_ops.mxfp4_quantize(b)[0], torch.bfloat16)
    want = hip_ops.mxfp4_gemm(hip_ops.mxfp4_quantize(a[-500:])[0], hip_ops.mxfp4_quantize(b[-700:])[0], torch.bfloat16)
    assert torch.equal(out[-500:, -700:], want)


def test_tokens_and_experts(device):
    tokens, top_k, experts, width, out_dim = 80000, 8, 16, 7168, 96
    gen = torch.Generator(device=device).manual_seed(2)
    ids = torch.randint(0, experts, (tokens, top_k), generator=gen, device=device)
    x = torch.randn(tokens, width, generator=gen, device=device, dtype=torch.bfloat16)
    routing = route_tokens(ids, experts)
    rows = dispatch_tokens(x, routing)
    source = routing.source[-1000:].long() // top_k
    assert torch.equal(rows[-1000:], x[source])
    back = combine_tokens(rows, routing, torch.full((tokens, top_k), 0.125, device=device))
    assert torch.equal(back[-1000:], x[-1000:])
    weight = torch.randn(experts, out_dim, width, generator=gen, device=device, dtype=torch.bfloat16)
    by_rows = mxfp4_expert_linear(rows, weight, routing, sorted_rows=True)
    assert torch.equal(by_rows, mxfp4_expert_linear(x, weight, routing))
    last = hip_ops.mxfp4_gemm(hip_ops.mxfp4_quantize(x[source])[0], hip_ops.mxfp4_quantize(weight[-1])[0], torch.bfloat16)
    # (other tiles can add the steps in another order: a rounding of the result, twice)
    assert (by_rows[-1000:].float() - last.float()).abs().max() <= 2.0**-7 * last.float().abs().max()
