"""Routings of tables that :func:`route_tokens` did not make: kernels index by them, so wrong ones are refused."""

import pytest
import torch

from flex_shard_amd.experts import ExpertRouting, combine_tokens, dispatch_tokens, route_tokens
from flex_shard_amd.mxfp4 import mxfp4_expert_linear


def tables(ids, experts):
    """position, offsets, source and padded offsets of choices [tokens, top_k], by sorting."""
    flat = torch.where((ids < 0) | (ids >= experts), experts, ids).flatten()
    order = torch.argsort(flat, stable=True)
    lengths = torch.bincount(flat, minlength=experts + 1)[:experts]
    offsets = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)])
    rank = torch.empty_like(order)
    rank[order] = torch.arange(len(order), device=ids.device)
    position = torch.where(flat < experts, rank, -1).view(ids.shape)
    source = torch.where(torch.arange(len(order), device=ids.device) < offsets[-1], order, -1)
    padded = torch.cat([lengths.new_zeros(1), ((lengths + 255) // 256 * 256).cumsum(0)])
    return [t.to(torch.int32) for t in (position, offsets, source, padded)]


IDS = torch.tensor([[0, 2], [2, -1], [1, 2], [7, 0]])


@pytest.mark.parametrize("ids,experts", [(IDS, 3), (IDS, 8), (torch.empty(0, 2, dtype=torch.int64), 3), (torch.full((300, 2), 1), 2),
                                         (torch.full((5, 1), -1), 2)])
def test_right_tables(ids, experts):
    routing = ExpertRouting(experts, *tables(ids, experts))
    routing.check()
    assert len(routing.pointers()) == 4
    again = ExpertRouting.of_buffer(experts, ids.shape, routing.buffer)
    again.check()


@pytest.mark.parametrize("dtype", [torch.int64, torch.float32, torch.int16])
def test_tables_of_another_type(dtype):
    for which in (slice(0, 4), slice(0, 1), slice(1, 2)):
        made = tables(IDS, 3)
        made[which] = [t.to(dtype) for t in made[which]]
        if torch.cat([t.flatten() for t in made]).dtype == torch.int32:
            continue  # (concatenated to int32 without a loss)
        routing = ExpertRouting(3, *made)
        for use in (routing.check, routing.pointers):
            with pytest.raises(ValueError, match="int32"):
                use()


def test_tables_of_other_sizes():
    made = tables(IDS, 3)
    with pytest.raises(ValueError, match="elements"):
        ExpertRouting(2, *made).pointers()
    position, offsets, source, padded = made
    # as many numbers in all, not in each
    with pytest.raises(ValueError, match="elements"):
        ExpertRouting(3, position, offsets[:-1], source, torch.cat([padded, padded[-1:]])).pointers()
    with pytest.raises(ValueError, match="elements"):
        ExpertRouting.of_buffer(3, IDS.shape, torch.cat([position.flatten(), source, offsets])).pointers()
    with pytest.raises(ValueError, match="1024"):
        ExpertRouting(1025, *tables(IDS, 1025)).pointers()
    with pytest.raises(ValueError, match="1024"):
        ExpertRouting(0, position, offsets[:1], source, padded[:1]).pointers()


# table (position, offsets, source, padded), place, value
@pytest.mark.parametrize(
    "table,at,value",
    [(0, 0, 8), (0, 0, -2), (0, 0, 1), (0, 3, 7), (0, 0, -1), (1, 0, 1), (1, 1, -1), (1, 1, 4), (1, 3, 9), (1, 3, 5), (2, 0, 8), (2, 0, -1),
     (2, 0, 1), (2, 7, 0), (3, 0, 256), (3, 1, 255), (3, 3, 512), (3, 3, 1 << 30)],
)
def test_tables_with_a_wrong_number(table, at, value):
    made = tables(IDS, 3)
    assert made[table].view(-1)[at] != value
    made[table].view(-1)[at] = value
    routing = ExpertRouting(3, *made)
    for use in (routing.check, routing.pointers):
        with pytest.raises(ValueError, match="order"):
            use()


@pytest.mark.gpu
def test_on_the_gpu(device):
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(-1, 9, (70, 3), generator=gen).to(device)
    made, by_hand = route_tokens(ids, 8), ExpertRouting(8, *tables(ids, 8))
    x, w = torch.randn(70, 64, device=device), torch.randn(8, 40, 64, device=device)
    weights = torch.rand(70, 3, device=device)
    results = []
    for routing in (made, by_hand):
        rows = dispatch_tokens(x, routing)
        results.append((rows, mxfp4_expert_linear(x, w, routing), combine_tokens(rows, routing, weights)))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert torch.equal(made.buffer, by_hand.buffer)
    wide = ExpertRouting(8, *[t.long() for t in tables(ids, 8)])
    for use in (lambda: dispatch_tokens(x, wide), lambda: combine_tokens(rows, wide, weights), lambda: mxfp4_expert_linear(x, w, wide),
                lambda: mxfp4_expert_linear(rows, w, wide, sorted_rows=True)):
        with pytest.raises(ValueError, match="int32"):
            use()
