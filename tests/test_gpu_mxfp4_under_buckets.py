"""4-bit layers and an expert stack whose parameters live in buckets: gathered for the forward and again for the backward,
their full storage freed in between.  Outputs and shard gradients equal the unsharded model's, bit for bit."""

import pytest
import torch
import torch.nn as nn

from flex_shard_amd import BucketedBlockShard, LocalReduceGroup
from flex_shard_amd.experts import combine_tokens, route_tokens
from flex_shard_amd.flex_shard import BucketCommContext, BucketRuntime
from flex_shard_amd.mxfp4 import convert_to_flex_shard_mxfp4_linear, mxfp4_expert_linear
from flex_shard_amd.testing import FakeMesh

pytestmark = pytest.mark.gpu


class _Experts(nn.Module):
    def __init__(self, experts: int, dim: int, hidden: int) -> None:
        super().__init__()
        self.up = nn.Parameter(torch.randn(experts, hidden, dim) * dim**-0.5)
        self.down = nn.Parameter(torch.randn(experts, dim, hidden) * hidden**-0.5)

    def forward(self, x):
        ids = torch.stack([torch.arange(len(x), device=x.device) % 3, torch.full((len(x),), 3, device=x.device)], dim=1)
        routing = route_tokens(ids, self.up.shape[0])
        rows = mxfp4_expert_linear(torch.relu(mxfp4_expert_linear(x, self.up, routing)), self.down, routing, sorted_rows=True)
        return combine_tokens(rows, routing, torch.full(ids.shape, 0.5, device=x.device))


def _model(device):
    torch.manual_seed(4)
    model = nn.Sequential(nn.Linear(256, 128, bias=False), _Experts(5, 128, 256), nn.Linear(128, 256, bias=False))
    return convert_to_flex_shard_mxfp4_linear(model.to(device, torch.bfloat16))


def test_dense_buckets(device):
    model, plain = _model(device), _model(device)
    context = BucketCommContext.create(device, max_pending_reduce_grads=1)
    mesh = FakeMesh(1, 0, LocalReduceGroup(1, 0))
    runtimes = []
    for layer, names in zip(model, (["0.weight"], ["1.up", "1.down"], ["2.weight"])):
        placement = BucketedBlockShard(dims=(0,), blocks_per_rank=(1,))
        runtime = BucketRuntime.shard_module_params(model, names, placement, mesh, context)
        runtime.install_hooks(layer)
        runtimes.append(runtime)
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(70, 256, generator=gen).bfloat16().to(device)
    grad_out = torch.randn(70, 256, generator=gen).bfloat16().to(device)
    for step in range(2):
        if step:  # an optimizer's step: the next gathering brings other values
            with torch.no_grad():
                for p in [p for r in runtimes for p in r.sharded_params] + list(plain.parameters()):
                    p.mul_(0.75)
        x_run, x_ref = x.clone().requires_grad_(), x.clone().requires_grad_()
        out = model(x_run)
        assert all(not r.is_unsharded for r in runtimes)
        assert all(b.untyped_storage().size() == 0 for r in runtimes for b in r.persistent_buffers)
        out.backward(grad_out)
        context.wait_and_clear_reduce_grad_states()
        ref = plain(x_ref)
        ref.backward(grad_out)
        assert torch.equal(out.detach(), ref.detach()) and torch.equal(x_run.grad, x_ref.grad)
        shards = [p for r in runtimes for p in r.sharded_params]
        for shard, full in zip(shards, plain.parameters(), strict=True):
            assert full.grad.any() and torch.equal(shard.grad.view(full.shape), full.grad)
            shard.grad = full.grad = None
    torch.cuda.synchronize()
