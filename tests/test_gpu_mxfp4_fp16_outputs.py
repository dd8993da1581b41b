"""fp16 results are the fp32 results rounded once, to nearest even, subnormal ones and ties included."""

import pytest
import torch

from flex_shard_amd import hip_ops
from flex_shard_amd.experts import combine_tokens, route_tokens

pytestmark = pytest.mark.gpu


def _same(got, want):
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan)
    assert torch.equal(got[~nan].view(torch.int16), want[~nan].view(torch.int16))


@pytest.mark.parametrize("width", [1024, 1023])
@pytest.mark.parametrize("weight", [0.5, 0.75, 1.0, 1.5, 0.0625, 2.0**-11, 0.3, 40000.0])
def test_every_value_weighted(device, width, weight):
    values = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)[: 64 * width].view(64, width).to(device)
    routing = route_tokens(torch.zeros(64, 1, dtype=torch.int64, device=device), 1)
    weights = torch.full((64, 1), weight, device=device)
    got = combine_tokens(values, routing, weights)
    # (a sum over the choices that starts from +0: a product of -0 gives +0)
    _same(got.cpu(), (0.0 + values.cpu().float() * torch.tensor(weight)).half())


@pytest.mark.parametrize("scale", [1.0, 2.0**-9, 2.0**-12, 2.0**9])
@pytest.mark.parametrize("m,n,k", [(1, 300, 512), (16, 264, 512), (70, 130, 256), (700, 1300, 512), (1500, 2048, 256), (4096, 4096, 256)])
def test_products(device, m, n, k, scale):
    gen = torch.Generator(device=device).manual_seed(m)
    a = hip_ops.mxfp4_quantize(torch.randn(m, k, generator=gen, device=device) * scale)[0]
    b = hip_ops.mxfp4_quantize(torch.randn(n, k, generator=gen, device=device) * scale)[0]
    exact = hip_ops.mxfp4_gemm(a, b, torch.float32)
    _same(hip_ops.mxfp4_gemm(a, b, torch.float16).cpu(), exact.cpu().half())
