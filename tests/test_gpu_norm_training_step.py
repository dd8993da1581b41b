"""Norms in 8 bits, FP8 linears, clipping and AdamW as a training step has them:
on sharded buckets under the runtime's hooks, every value the bits of the same step
without sharding and with the norm in bf16."""

import pytest
import torch
import torch.nn as nn
from torch.nn import functional as F

from flex_shard_amd import BucketedBlockShard, Fp8BucketedBlockShard, LocalReduceGroup, get_global_layout
from flex_shard_amd.adamw import FlexShardAdamW, grad_square_sum
from flex_shard_amd.blockwise_fp8 import (
    BlockwiseFp8Weight, convert_to_flex_shard_float8_blockwise_linear, make_blockwise_fp8_weight, prequantized_linear,
)
from flex_shard_amd.custom_placements.fp8_bucketed_block_shard import _quantize_dense_weight_to_blockwise_fp8
from flex_shard_amd.dist_muon import OwnedMuon
from flex_shard_amd.flex_shard import BucketCommContext, BucketRuntime, register_optimizer_checkpoint_hook
from flex_shard_amd.norms import FlexShardRMSNorm, convert_to_flex_shard_rms_norm, rms_norm
from flex_shard_amd.testing import FakeMesh

pytestmark = pytest.mark.gpu

DIM, HIDDEN, TOKENS = 256, 384, 70
HYPER = dict(lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1)


class _Mlp(nn.Module):
    def __init__(self):
        super().__init__()
        self.gate, self.up = nn.Linear(DIM, HIDDEN, bias=False), nn.Linear(DIM, HIDDEN, bias=False)
        self.down = nn.Linear(HIDDEN, DIM, bias=False)

    def forward(self, a):
        return self.down(F.silu(self.gate(a)) * self.up(a))


class _Block(nn.Module):
    def __init__(self):
        super().__init__()
        self.norm, self.mlp = nn.RMSNorm(DIM, eps=1e-6), _Mlp()

    def forward(self, x, stream):
        a, stream = self.norm(x, stream, fp8=True)
        return self.mlp(a), stream


def _model(device):
    torch.manual_seed(7)
    model = nn.ModuleList([_Block(), _Block()]).to(device, torch.bfloat16)
    for block in model:
        nn.init.normal_(block.norm.weight, 1.0, 0.1)
    return model


def _reference(params, x, grad_out, grad_stream):
    """Output, stream and gradients of the two blocks without sharding."""
    leaves = {}
    for name, p in params.items():
        if "norm" in name:
            leaves[name] = p.detach().clone().requires_grad_()
        else:
            q, s = _quantize_dense_weight_to_blockwise_fp8(p.detach(), 128, torch.float8_e4m3fn)
            leaves[name] = BlockwiseFp8Weight(q, s, 128, requires_grad=True)
    y, stream = x, torch.zeros_like(x, dtype=torch.float32)
    for i in range(2):
        a, stream = rms_norm(y, leaves[f"{i}.norm.weight"], 1e-6, residual=stream)
        gate, up = (prequantized_linear(a, leaves[f"{i}.mlp.{part}.weight"]) for part in ("gate", "up"))
        y = prequantized_linear(F.silu(gate) * up, leaves[f"{i}.mlp.down.weight"])
    grads = torch.autograd.grad([y, stream], list(leaves.values()), [grad_out, grad_stream])
    return y.detach(), stream.detach(), dict(zip(leaves, grads))


@pytest.mark.parametrize("bits", [32, 8])
def test_sharded_step(device, bits):
    model = _model(device)
    full = {name: nn.Parameter(p.detach().clone()) for name, p in model.named_parameters()}
    convert_to_flex_shard_rms_norm(model)
    convert_to_flex_shard_float8_blockwise_linear(model)
    assert type(model[0].norm) is FlexShardRMSNorm
    context = BucketCommContext.create(device)
    mesh = FakeMesh(1, 0, LocalReduceGroup(1, 0))
    runtimes = []
    for i, block in enumerate(model):
        # (the norm's bucket is resharded before the linears' is unsharded)
        norm = BucketRuntime.shard_module_params(
            model, [f"{i}.norm.weight"], BucketedBlockShard(dims=(0,), blocks_per_rank=(1,)), mesh, context
        )
        linears = BucketRuntime.shard_module_params(
            model, [f"{i}.mlp.{part}.weight" for part in ("gate", "up", "down")],
            Fp8BucketedBlockShard(world_size=1, weight_factory=make_blockwise_fp8_weight), mesh, context,
        )
        norm.install_hooks(block.norm)
        linears.install_hooks(block.mlp)
        runtimes += [norm, linears]
    shards = {bp.info.fqn: bp.sharded_param for r in runtimes for bp in r.bucket_params}
    optimizer = FlexShardAdamW(shards.values(), **HYPER, state_bits=bits)
    twin = FlexShardAdamW([full[name] for name in shards], **HYPER, state_bits=bits)
    gen = torch.Generator(device=device).manual_seed(3)
    for step in range(3):
        x = torch.randn(TOKENS, DIM, generator=gen, device=device).bfloat16()
        grad_out = (torch.randn(TOKENS, DIM, generator=gen, device=device) * 0.1).bfloat16()
        grad_stream = torch.randn(TOKENS, DIM, generator=gen, device=device) * 0.1
        y, stream = x, torch.zeros_like(x, dtype=torch.float32)
        for block in model:
            y, stream = block(y, stream)
        assert all(b.untyped_storage().size() == 0 for r in runtimes for b in r.persistent_buffers)
        torch.autograd.backward([y, stream], [grad_out, grad_stream])
        context.wait_and_clear_reduce_grad_states()
        want_y, want_stream, grads = _reference(full, x, grad_out, grad_stream)
        assert torch.equal(y.detach(), want_y) and torch.equal(stream.detach(), want_stream)
        for name, shard in shards.items():
            assert grads[name].any() and torch.equal(shard.grad.view(grads[name].shape), grads[name].to(shard.grad.dtype)), name
            full[name].grad = shard.grad.view(full[name].shape).clone()
        for o, ps in ((optimizer, shards.values()), (twin, full.values())):
            o.step(square_sum=grad_square_sum([p.grad for p in ps]), max_norm=1.0)
        for name, shard in shards.items():
            assert torch.equal(shard.view(full[name].shape), full[name]), name
            shard.grad = None
    torch.cuda.synchronize()


def test_states_get_their_shards_layouts(device):
    model = _model(device)
    context = BucketCommContext.create(device)
    runtime = BucketRuntime.shard_module_params(
        model, ["0.norm.weight", "1.norm.weight"], BucketedBlockShard(dims=(0,), blocks_per_rank=(1, 1)), FakeMesh(2, 0, LocalReduceGroup(2, 0)), context
    )
    shards = runtime.sharded_params
    for p in shards:
        p.grad = torch.ones_like(p)
    optimizer = FlexShardAdamW(shards)
    register_optimizer_checkpoint_hook(optimizer, [runtime])
    optimizer.step()
    state = optimizer.state_dict()["state"]
    for name in ("exp_avg", "exp_avg_sq"):
        layout = get_global_layout(state[0][name])
        assert tuple(layout.global_shape) == (DIM,) and sum(s[0] for s in layout.local_sizes) == shards[0].numel()
    assert get_global_layout(state[0]["step"]) is None
    eight = FlexShardAdamW(shards, state_bits=8)
    register_optimizer_checkpoint_hook(eight, [runtime])
    eight.step()
    with pytest.raises(NotImplementedError, match="scale"):  # a scale covers 128 elements of this rank's shard
        eight.state_dict()


def test_a_resharded_weight_is_refused(device):
    norm = FlexShardRMSNorm(DIM, device=device, dtype=torch.bfloat16)
    x = torch.zeros(3, DIM, dtype=torch.bfloat16, device=device)
    freed = torch.zeros_like(x)
    freed.untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="residual has no memory"):
        norm(x, freed)
    norm.weight.untyped_storage().resize_(0)
    for fp8 in (False, True):
        with pytest.raises(RuntimeError, match="resharded"):
            norm(x, fp8=fp8)
    p = nn.Parameter(torch.zeros(5, device=device))
    p.grad = torch.ones_like(p)
    p.untyped_storage().resize_(0)
    with pytest.raises(RuntimeError, match="null pointer"):
        FlexShardAdamW([p]).step()


def test_beside_muon(device):
    """Matrices by Muon, the rest by AdamW, as one step; each as it would be alone."""
    model, twin = _model(device), _model(device)
    convert_to_flex_shard_rms_norm(model)

    def split(m):
        return [p for p in m.parameters() if p.ndim == 2], [p for p in m.parameters() if p.ndim == 1]

    matrices, vectors = split(model)
    muon, adamw = OwnedMuon(matrices, lr=0.01), FlexShardAdamW(vectors, **HYPER)
    matrices_alone, vectors_alone = split(twin)
    muon_alone = OwnedMuon(matrices_alone, lr=0.01)
    adamw_alone = [FlexShardAdamW([p], **HYPER) for p in vectors_alone]
    gen = torch.Generator(device=device).manual_seed(4)
    for _ in range(2):
        x = torch.randn(TOKENS, DIM, generator=gen, device=device).bfloat16()
        y = x
        for block in model:
            y = y + block.mlp(block.norm(y))
        y.float().square().mean().backward()
        for p, q in zip(matrices + vectors, matrices_alone + vectors_alone):
            q.grad = p.grad.clone()
        muon.step([p.grad for p in matrices])
        adamw.step()
        for o in adamw_alone:
            o.step()
        muon_alone.step([p.grad for p in matrices_alone])
        for p, q in zip(matrices + vectors, matrices_alone + vectors_alone):
            assert torch.equal(p, q)
        model.zero_grad()
