"""Tokens sorted by expert and back, against counting and float64 sums."""

import numpy as np
import pytest
import torch
from mxfp4_definition import ROUNDING

from flex_shard_amd import hip_ops
from flex_shard_amd.experts import combine_tokens, dispatch_tokens, route_tokens

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _ids(tokens, top_k, experts, seed, here=1.0):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, experts, (tokens, top_k), generator=gen)
    away = torch.rand(tokens, top_k, generator=gen) >= here
    return torch.where(away, torch.where(ids % 3 == 0, -1 - ids, experts + ids), ids)


def _assert_sorted(routing, ids, experts):
    flat = ids.flatten().numpy()
    source = np.concatenate([np.flatnonzero(flat == e) for e in range(experts)])
    counts = np.array([(flat == e).sum() for e in range(experts)])
    position = np.full(flat.shape, -1)
    position[source] = np.arange(len(source))
    assert np.array_equal(routing.offsets.cpu().numpy(), np.concatenate([[0], counts.cumsum()]))
    assert np.array_equal(routing.padded_offsets.cpu().numpy(), np.concatenate([[0], (-(-counts // 256) * 256).cumsum()]))
    assert int(routing.padded_offsets[-1]) <= routing.padded_rows
    assert np.array_equal(routing.position.cpu().numpy().ravel(), position)
    assert np.array_equal(routing.source.cpu().numpy(), np.concatenate([source, np.full(len(flat) - len(source), -1)]))
    assert all(t.dtype == torch.int32 for t in (routing.position, routing.offsets, routing.source, routing.padded_offsets))


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
@pytest.mark.parametrize(
    "tokens,top_k,experts,here",
    [(1, 1, 1, 1.0), (1, 8, 256, 1.0), (7, 3, 2, 0.5), (256, 8, 64, 1.0), (257, 8, 63, 0.9), (1000, 2, 5, 0.0), (3001, 1, 1, 1.0),
     (5000, 8, 257, 0.3), (777, 6, 1024, 1.0)],
)
def test_route(device, tokens, top_k, experts, here, dtype):
    ids = _ids(tokens, top_k, experts, tokens, here)
    _assert_sorted(route_tokens(ids.to(device, dtype), experts), ids, experts)


def test_route_of_one_expert_of_strided_ids_and_of_ids_beyond_32_bits(device):
    ids = torch.full((2500, 4), 2)
    _assert_sorted(route_tokens(ids.to(device), 3), ids, 3)
    wide = _ids(300, 8, 16, 3)
    _assert_sorted(route_tokens(wide.to(device)[:, ::2], 16), wide[:, ::2], 16)
    _assert_sorted(route_tokens(wide.to(device).t(), 16), wide.t().contiguous(), 16)
    far = wide + torch.where(wide % 2 == 0, 1 << 32, 0)
    _assert_sorted(route_tokens(far.to(device), 16), far, 16)


WIDTHS = [(1, 1, 1), (1, 8, 7168), (5, 2, 64), (33, 3, 1001), (64, 64, 24), (300, 6, 2056)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,top_k,width", WIDTHS)
def test_rows_there_and_back(device, tokens, top_k, width, dtype):
    experts = 9
    ids = _ids(tokens, top_k, experts, 1, 0.8)
    if tokens > 2:
        ids[1] = -1  # a token none of whose experts are here
    routing = route_tokens(ids.to(device), experts)
    gen = torch.Generator().manual_seed(2)
    x, g = (torch.randn(tokens, width, generator=gen).to(dtype) for _ in range(2))
    rows, g_sorted = (torch.randn(tokens * top_k, width, generator=gen).to(dtype) for _ in range(2))
    position, used = routing.position.cpu().long(), int(routing.offsets[-1])
    rows[used:], g_sorted[used:] = float("nan"), float("inf")  # rows of no expert are never read
    here, at = (position >= 0)[..., None], position.clamp(min=0)
    u = ROUNDING[dtype]
    tiny = 2.0**-25 if dtype == torch.float16 else 2.0**-133

    x_leaf = x.to(device).requires_grad_()
    gathered = dispatch_tokens(x_leaf, routing)
    want = torch.zeros(tokens * top_k, width, dtype=dtype)
    want[position[position >= 0]] = x[:, None].expand(-1, top_k, -1)[position >= 0]
    assert torch.equal(gathered.cpu(), want)
    (gx,) = torch.autograd.grad(gathered, x_leaf, g_sorted.to(device))
    parts = torch.where(here, g_sorted.double()[at], 0.0)
    assert ((gx.double().cpu() - parts.sum(1)).abs() <= top_k * 2.0**-24 * parts.abs().sum(1) + u * parts.sum(1).abs() + tiny).all()

    for weights_dtype in (torch.float32, dtype):
        weights = torch.rand(tokens, top_k, generator=gen).to(weights_dtype)
        leaves = [rows.to(device).requires_grad_(), weights.to(device).requires_grad_()]
        back = combine_tokens(leaves[0], routing, leaves[1])
        assert back.dtype == dtype
        parts = torch.where(here, rows.double()[at], 0.0) * weights.double()[..., None]
        assert ((back.double().cpu() - parts.sum(1)).abs() <= (top_k + 1) * 2.0**-24 * parts.abs().sum(1) + u * parts.sum(1).abs() + tiny).all()
        if tokens > 2:
            assert not back[1].any()
        g_rows, g_weights = torch.autograd.grad(back, leaves, g.to(device))
        assert g_rows.dtype == dtype and g_weights.dtype == weights_dtype
        want_rows = torch.zeros(tokens * top_k, width, dtype=torch.float64)
        want_rows[position[position >= 0]] = (weights.double()[..., None] * g.double()[:, None])[position >= 0]
        assert ((g_rows.double().cpu() - want_rows).abs() <= (u + 2.0**-24) * want_rows.abs() + tiny).all()
        products = torch.where(here, rows.double()[at] * g.double()[:, None], 0.0)
        error = (g_weights.double().cpu() - products.sum(-1)).abs()
        smallest = 2.0**-25 if weights_dtype == torch.float16 else 0.0
        assert (error <= (width + 8) * 2.0**-24 * products.abs().sum(-1) + ROUNDING[weights_dtype] * products.sum(-1).abs() + smallest).all()
        assert not g_weights.cpu()[position < 0].any()


def test_combine_against_differences(device):
    """The weighted sum is linear in its rows and in its weights: a step of either
    changes the loss by the gradient times the step, up to the sums' rounding."""
    ids = _ids(20, 3, 4, 5, 0.8)
    routing = route_tokens(ids.to(device), 4)
    gen = torch.Generator().manual_seed(1)
    rows, weights, g = torch.randn(60, 40, generator=gen).to(device), torch.rand(20, 3, generator=gen).to(device), torch.randn(20, 40, generator=gen)

    def loss(rows, weights):
        return (combine_tokens(rows, routing, weights).cpu().double() * g.double()).sum().item()

    leaves = [rows.clone().requires_grad_(), weights.clone().requires_grad_()]
    g_rows, g_weights = torch.autograd.grad(combine_tokens(leaves[0], routing, leaves[1]), leaves, g.to(device))
    base, used = loss(rows, weights), int(routing.offsets[-1])
    # a sum of three products of size 1 is off by 2**-22 at most, times 40 gradients of size 4 at most
    slack = 2 * 40 * 4 * 2.0**-21
    for r in (0, used // 2, used - 1):
        moved = rows.clone()
        moved[r, 7] += 0.5
        assert abs(loss(moved, weights) - base - 0.5 * g_rows[r, 7].item()) <= slack
    for t, j in ((0, 0), (7, 2), (19, 1)):
        moved = weights.clone()
        moved[t, j] += 0.5
        assert abs(loss(rows, moved) - base - 0.5 * g_weights[t, j].item()) <= slack


def test_results_are_the_same_every_time(device):
    ids = _ids(4000, 8, 32, 7).to(device)
    gen = torch.Generator(device=device).manual_seed(1)
    rows = torch.randn(32000, 264, generator=gen, device=device)
    first = None
    for _ in range(3):
        routing = route_tokens(ids, 32)
        grads = hip_ops.expert_combine_backward(rows[:4000].contiguous(), rows, routing.position, routing.offsets,
                                                torch.ones(4000, 8, device=device))
        now = (routing.position, routing.source, hip_ops.expert_combine(rows, routing.position), *grads)
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


def test_no_tokens_and_no_width(device):
    routing = route_tokens(torch.empty(0, 4, dtype=torch.int64, device=device), 3)
    assert routing.offsets.tolist() == routing.padded_offsets.tolist() == [0, 0, 0, 0] and routing.rows == 0
    x = torch.empty(0, 16, device=device, requires_grad=True)
    gathered = dispatch_tokens(x, routing)
    back = combine_tokens(gathered, routing, torch.empty(0, 4, device=device))
    assert gathered.shape == back.shape == (0, 16)
    back.sum().backward()
    assert x.grad.shape == (0, 16)
    routing = route_tokens(torch.zeros(3, 2, dtype=torch.int64, device=device), 1)
    weights = torch.ones(3, 2, device=device, requires_grad=True)
    combine_tokens(torch.empty(6, 0, device=device), routing, weights).sum().backward()
    assert torch.equal(weights.grad, torch.zeros(3, 2, device=device))


def test_refusals(device):
    ids = torch.zeros(4, 2, dtype=torch.int64, device=device)
    with pytest.raises(RuntimeError, match="no CPU path"):
        route_tokens(ids.cpu(), 3)
    with pytest.raises(ValueError, match="int64 or int32"):
        route_tokens(ids.float(), 3)
    with pytest.raises(ValueError, match="at least one"):
        route_tokens(ids, 0)
    with pytest.raises(Exception, match="1024"):
        route_tokens(ids, 1025)
    with pytest.raises(ValueError, match="top_k"):
        route_tokens(ids[0], 3)
    routing = route_tokens(ids, 3)
    with pytest.raises(ValueError, match="x must be"):
        dispatch_tokens(torch.zeros(5, 8, device=device), routing)
    with pytest.raises(ValueError, match="rows must be"):
        combine_tokens(torch.zeros(4, 8, device=device), routing, torch.ones(4, 2, device=device))
    with pytest.raises(ValueError, match="weights must be"):
        combine_tokens(torch.zeros(8, 8, device=device), routing, torch.ones(4, 1, device=device))
    with pytest.raises(NotImplementedError):
        dispatch_tokens(torch.zeros(4, 8, device=device, dtype=torch.float64), routing)
    many = route_tokens(torch.zeros(2, 65, dtype=torch.int64, device=device), 3)
    with pytest.raises(Exception, match="at most 64"):
        dispatch_tokens(torch.zeros(2, 8, device=device), many)
