"""The entries that take a routing's tables, and a quantized matrix's data and scales, as tensors."""

import pytest
import torch

from flex_shard_amd import hip_ops
from flex_shard_amd.experts import combine_tokens, dispatch_tokens, route_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_tables_are_those_of_a_routing(device, dtype):
    gen = torch.Generator(device=device).manual_seed(1)
    ids = torch.randint(-1, 9, (300, 3), generator=gen, device=device).to(dtype)
    routing = route_tokens(ids, 8)
    position, offsets, source, padded_offsets = hip_ops.expert_route(ids, 8)
    for got, want in ((position, routing.position), (offsets, routing.offsets), (source, routing.source), (padded_offsets, routing.padded_offsets)):
        assert got.dtype == torch.int32 and torch.equal(got, want)
    x = torch.randn(300, 72, generator=gen, device=device)
    rows = hip_ops.expert_dispatch(x, position, offsets)
    assert torch.equal(rows, dispatch_tokens(x, routing))
    weights = torch.rand(300, 3, generator=gen, device=device)
    assert torch.equal(hip_ops.expert_combine(rows, position, weights), combine_tokens(rows, routing, weights))


def test_refusals(device):
    ids = torch.zeros(4, 2, dtype=torch.int64, device=device)
    position, offsets, source, _ = hip_ops.expert_route(ids, 3)
    x = torch.zeros(4, 8, device=device)
    with pytest.raises(ValueError, match="position"):
        hip_ops.expert_dispatch(x, position.long(), offsets)
    with pytest.raises(ValueError, match="position"):
        hip_ops.expert_dispatch(x[:3], position, offsets)
    with pytest.raises(ValueError, match="offsets"):
        hip_ops.expert_dispatch(x, position, offsets.long())
    with pytest.raises(ValueError, match="x must be"):
        hip_ops.expert_dispatch(torch.zeros(4, 16, device=device)[:, ::2], position, offsets)
    with pytest.raises(RuntimeError, match="no CPU path"):
        hip_ops.expert_dispatch(x, position.cpu(), offsets)
    with pytest.raises(NotImplementedError, match="own type"):
        hip_ops.expert_combine_at(torch.zeros(8, 8, device=device, dtype=torch.bfloat16), position.data_ptr(), 4, 2, dtype=torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("left,cols", [(0, 300), (8, 296), (3, 257)])
def test_dequantize_into_rows_of_a_wider_matrix(device, left, cols, dtype):
    gen = torch.Generator(device=device).manual_seed(cols)
    matrix = hip_ops.mxfp4_quantize(torch.randn(37, cols, generator=gen, device=device))[0]
    wide = torch.full((37, 320), 7.0, dtype=dtype, device=device)
    out = hip_ops.mxfp4_dequantize(*matrix, cols, dtype, out=wide[:, left : left + cols])
    want = matrix.dequantize(dtype)
    assert torch.equal(out, want) and torch.equal(hip_ops.mxfp4_dequantize(matrix.data, matrix.scales, cols, dtype), want)
    assert (wide[:, :left] == 7.0).all() and (wide[:, left + cols :] == 7.0).all()
