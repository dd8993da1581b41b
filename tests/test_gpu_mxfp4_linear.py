"""Products, linear layers and experts' layers on 4-bit operands against float64
products of the values that the operands stand for."""

import pytest
import torch
import torch.nn as nn
from mxfp4_definition import ROUNDING, assert_product, through

from flex_shard_amd import _native, hip_ops
from flex_shard_amd.experts import combine_tokens, dispatch_tokens, route_tokens
from flex_shard_amd.mxfp4 import (
    FlexShardMxFp4Linear,
    convert_to_flex_shard_mxfp4_linear,
    mxfp4_expert_linear,
    mxfp4_linear,
    mxfp4_quantize,
    quantize_mxfp4_weight,
)

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
# tokens, out, in: single tokens, fewer and more rows than any tile, sizes that end inside tiles and runs
SIZES = [(1, 1, 1), (1, 130, 96), (2, 64, 256), (5, 1000, 320), (16, 96, 4096), (17, 48, 512), (33, 257, 1000), (64, 64, 31),
         (100, 513, 2048), (128, 128, 128), (257, 300, 700), (520, 777, 290), (1100, 1030, 640)]


def _normal(shape, scale, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("tokens,out_dim,in_dim", SIZES)
def test_forward(device, tokens, out_dim, in_dim, bias, dtype):
    x, w = _normal((tokens, in_dim), 1.0, dtype, 1), _normal((out_dim, in_dim), 0.05, dtype, 2)
    b = _normal((out_dim,), 1.0, dtype, 3) if bias else None
    on_gpu = None if b is None else b.to(device)
    got = mxfp4_linear(x.to(device), w.to(device), on_gpu)
    assert got.dtype == dtype
    assert_product(got, through(x), through(w), None if b is None else b.double())
    with torch.no_grad():
        served = mxfp4_linear(x.to(device), quantize_mxfp4_weight(w.to(device)), on_gpu)
    assert torch.equal(got, served)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,out_dim,in_dim", [(1, 1, 1), (3, 130, 96), (33, 257, 1000), (257, 300, 700), (1100, 530, 640)])
def test_gradients(device, tokens, out_dim, in_dim, dtype):
    x, w, b = _normal((tokens, in_dim), 1.0, dtype, 1), _normal((out_dim, in_dim), 0.05, dtype, 2), _normal((out_dim,), 1.0, dtype, 3)
    g = _normal((tokens, out_dim), 0.01, dtype, 4)
    leaves = [t.to(device).requires_grad_() for t in (x, w, b)]
    gx, gw, gb = torch.autograd.grad(mxfp4_linear(*leaves), leaves, g.to(device))
    assert_product(gx, through(g), through(w.t()))
    assert_product(gw, through(g.t()), through(x.t()))
    want, size = g.double().sum(dim=0), g.double().abs().sum(dim=0)
    smallest = 2.0**-25 if dtype == torch.float16 else 0.0
    assert ((gb.double().cpu() - want).abs() <= tokens * 2.0**-24 * size + ROUNDING[dtype] * want.abs() + smallest).all()
    # one gradient at a time gives the same
    for i, leaf in enumerate(leaves):
        others = [t.detach() for t in leaves]
        others[i] = leaf
        (alone,) = torch.autograd.grad(mxfp4_linear(*others), leaf, g.to(device))
        assert torch.equal(alone, (gx, gw, gb)[i])


# every kernel of the dense product: sizes that end inside its tiles, contractions of few and of many steps,
# more tiles than the chip holds at a time (256 x 256: a workgroup takes several)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize(
    "tiles,m,n,k",
    [("few rows", 4, 14340, 700), ("few rows", 16, 1001, 5000), ("64", 50, 3001, 1100), ("64", 300, 2048, 2048), ("128", 1000, 5123, 600),
     ("128", 8192, 1024, 1024), ("128 deep", 2040, 2040, 2300), ("128 deep", 2035, 2041, 700), ("256", 7950, 4096, 200),
     ("256", 8190, 4088, 520), ("256", 8001, 4091, 1030), ("256", 4090, 8192, 1792)],
)
def test_every_kernel(device, tiles, m, n, k, dtype):
    assert hip_ops.mxfp4_gemm_tiles(m, n, k) == tiles
    gen = torch.Generator(device=device).manual_seed(m + n)
    x, w = (torch.randn(rows, k, generator=gen, device=device).to(dtype) for rows in (m, n))
    a, b = mxfp4_quantize(x), mxfp4_quantize(w)
    bias = torch.randn(n, generator=gen, device=device).to(dtype)
    got = hip_ops.mxfp4_gemm(a, b, dtype, bias=bias)
    assert torch.equal(got, hip_ops.mxfp4_gemm(a, b, dtype, bias=bias))
    a64, b64 = a.dequantize(torch.float32).double(), b.dequantize(torch.float32).double()
    want, size = torch.mm(a64, b64.t()) + bias.double(), torch.mm(a64.abs(), b64.abs().t()) + bias.double().abs()
    assert ((got.double() - want).abs() <= (k + 1) * 2.0**-23 * size + ROUNDING[dtype] * want.abs()).all()
    # rows of a wider output, and nothing beside them
    wide = torch.full((m, n + 24), 7.0, dtype=dtype, device=device)
    assert torch.equal(hip_ops.mxfp4_gemm(a, b, dtype, bias=bias, out=wide[:, 5 : n + 5]), got)
    assert (wide[:, :5] == 7.0).all() and (wide[:, n + 5 :] == 7.0).all()


def test_fp32_master_weight_and_bias_with_bf16_activations(device):
    x, w, b = _normal((40, 96), 1.0, torch.bfloat16, 1), _normal((70, 96), 0.05, torch.float32, 2), _normal((70,), 1.0, torch.float32, 3)
    g = _normal((40, 70), 0.01, torch.bfloat16, 4)
    leaves = [t.to(device).requires_grad_() for t in (x, w, b)]
    y = mxfp4_linear(*leaves)
    assert y.dtype == torch.bfloat16
    assert_product(y, through(x), through(w), b.bfloat16().double())
    gx, gw, gb = torch.autograd.grad(y, leaves, g.to(device))
    assert gx.dtype == torch.bfloat16 and gw.dtype == gb.dtype == torch.float32
    assert_product(gw, through(g.t()), through(x.t()))


def _grid(shape, seed):
    """Values that quantize to themselves, along rows and columns: among the
    elements' own, with a 4 or a 6 in every run."""
    gen = torch.Generator().manual_seed(seed)
    values = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0])
    x = values[torch.randint(0, 6, shape, generator=gen)] * (1 - 2 * torch.randint(0, 2, shape, generator=gen))
    rows, cols = shape
    r, c = torch.arange(rows)[:, None], torch.arange(cols)[None]
    return torch.where((r + c) % 8 == 0, torch.where((r * c) % 2 == 0, 4.0, -6.0), x)


def test_gradients_against_differences(device):
    """Where the quantizers leave x and W as they are the layer is bilinear, and a
    step to another such value changes the loss by the gradient times the step."""
    tokens, out_dim, in_dim = 64, 32, 96
    x, w, g = _grid((tokens, in_dim), 1), _grid((out_dim, in_dim), 2), _grid((tokens, out_dim), 3)
    for t in (x, w, g):
        assert torch.equal(through(t), t.double()) and torch.equal(through(t.t()), t.t().double())

    def loss(x, w):
        return (mxfp4_linear(x.to(device), w.to(device)).double().cpu() * g.double()).sum().item()

    leaves = [t.to(device).requires_grad_() for t in (x, w)]
    gx, gw = torch.autograd.grad(mxfp4_linear(*leaves), leaves, g.to(device))
    base = loss(x, w)
    for at in ((0, 1), (13, 50), (63, 95)):
        moved = x.clone()
        moved[at] = 2.0 if x[at] != 2.0 else 1.0
        assert loss(moved, w) - base == (moved[at] - x[at]).item() * gx[at].item()
    for at in ((0, 1), (13, 50), (31, 94)):
        moved = w.clone()
        moved[at] = 2.0 if w[at] != 2.0 else 1.0
        assert loss(x, moved) - base == (moved[at] - w[at]).item() * gw[at].item()


def test_leading_dimensions_strides_and_empty_inputs(device):
    w = _normal((70, 96), 0.05, torch.bfloat16, 2).to(device).requires_grad_()
    wide = _normal((2, 3, 120), 1.0, torch.bfloat16, 1).to(device)
    x = wide[..., 7:103].detach().requires_grad_()
    y = mxfp4_linear(x, w)
    assert y.shape == (2, 3, 70)
    assert torch.equal(y.reshape(6, 70), mxfp4_linear(x.reshape(6, 96).contiguous(), w))
    gx, gw = torch.autograd.grad(y, (x, w), torch.ones((), dtype=torch.bfloat16, device=device).expand_as(y))  # a broadcast gradient
    assert gx.shape == x.shape and gw.shape == w.shape
    assert_product(gw, torch.ones(70, 6, dtype=torch.float64), through(x.detach().reshape(6, 96).t()))
    none = mxfp4_linear(x[:0], w)
    assert none.shape == (0, 3, 70)
    assert torch.equal(torch.autograd.grad(none.sum(), w)[0], torch.zeros_like(w))
    one = mxfp4_linear(x[0, 0], w)
    assert one.shape == (70,) and torch.equal(one, y[0, 0])


def test_nan_and_infinity_reach_their_rows_alone(device):
    x, w = _normal((40, 128), 1.0, torch.bfloat16, 1), _normal((70, 128), 0.05, torch.bfloat16, 2)
    clean = mxfp4_linear(x.to(device), w.to(device))
    x[3, 5], x[17, 100], w[9, 64] = float("nan"), float("inf"), -float("inf")
    got = mxfp4_linear(x.to(device), w.to(device))
    touched = torch.zeros(40, 70, dtype=torch.bool, device=device)
    touched[3], touched[17], touched[:, 9] = True, True, True
    assert torch.isnan(got[touched]).all() and torch.equal(got[~touched], clean[~touched])


def test_scales_of_zero_runs_and_very_different_runs(device):
    x, w = _normal((20, 256), 1.0, torch.float32, 1), _normal((24, 256), 1.0, torch.float32, 2)
    x[:, 32:64] = 0.0
    x[:, 64:96] *= 2.0**60
    w[:, 64:96] *= 2.0**-60
    x[4] = 0.0
    w[5, :128] = 0.0
    assert_product(mxfp4_linear(x.to(device), w.to(device)), through(x), through(w))


def test_frozen_weight(device):
    x, w = _normal((40, 96), 1.0, torch.bfloat16, 1).to(device).requires_grad_(), _normal((70, 96), 0.05, torch.bfloat16, 2)
    g = _normal((40, 70), 0.01, torch.bfloat16, 4)
    y = mxfp4_linear(x, quantize_mxfp4_weight(w.to(device), transposed=True))
    (gx,) = torch.autograd.grad(y, x, g.to(device))
    assert_product(gx, through(g), through(w.t()))
    with pytest.raises(RuntimeError, match="transposed"):
        mxfp4_linear(x, quantize_mxfp4_weight(w.to(device)))


def test_module_conversion(device):
    net = nn.Sequential(nn.Linear(64, 96), nn.ReLU(), nn.Sequential(nn.Linear(96, 32, bias=False))).to(device, torch.bfloat16)
    first, second = net[0].weight, net[2][0].weight
    convert_to_flex_shard_mxfp4_linear(net, lambda fqn, mod: fqn != "0")
    assert type(net[0]) is nn.Linear and isinstance(net[2][0], FlexShardMxFp4Linear) and net[2][0].weight is second
    convert_to_flex_shard_mxfp4_linear(net)
    assert isinstance(net[0], FlexShardMxFp4Linear) and net[0].weight is first
    x = torch.randn(10, 64, device=device, dtype=torch.bfloat16)
    out = net(x)
    out.sum().backward()
    assert out.shape == (10, 32) and all(p.grad is not None and torch.isfinite(p.grad).all() for p in net.parameters())


# ------------------------------------------------------------------- experts
def _ids(tokens, top_k, experts, seed, kind):
    gen = torch.Generator().manual_seed(seed)
    if kind == "one expert":
        return torch.full((tokens, top_k), experts - 1)
    ids = torch.randint(0, experts, (tokens, top_k), generator=gen)
    if kind == "few here":
        ids = torch.where(torch.rand(tokens, top_k, generator=gen) < 0.7, torch.where(ids % 2 == 0, -1, experts + 3), ids)
    if kind == "none here":
        ids = torch.full((tokens, top_k), -1)
    return ids


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sorted_rows", [False, True])
@pytest.mark.parametrize(
    "tokens,top_k,experts,out_dim,in_dim,kind",
    [(1, 1, 1, 16, 32, "random"), (1, 8, 32, 96, 320, "random"), (5, 2, 4, 130, 96, "few here"), (33, 3, 7, 65, 257, "random"),
     (64, 2, 5, 64, 64, "one expert"), (40, 2, 70, 48, 100, "random"), (16, 2, 3, 32, 64, "none here"), (700, 2, 3, 300, 290, "few here")],
)
def test_experts(device, tokens, top_k, experts, out_dim, in_dim, kind, sorted_rows, dtype):
    ids = _ids(tokens, top_k, experts, 5, kind)
    rows = tokens * top_k
    x, w = _normal((rows if sorted_rows else tokens, in_dim), 1.0, dtype, 1), _normal((experts, out_dim, in_dim), 0.05, dtype, 2)
    g = _normal((rows, out_dim), 0.01, dtype, 3)
    routing = route_tokens(ids.to(device), experts)
    leaves = [t.to(device).requires_grad_() for t in (x, w)]
    y = mxfp4_expert_linear(*leaves, routing, sorted_rows=sorted_rows)
    gx, gw = torch.autograd.grad(y, leaves, g.to(device))
    with torch.no_grad():
        served = mxfp4_expert_linear(leaves[0], quantize_mxfp4_weight(leaves[1]), routing, sorted_rows=sorted_rows)
    assert torch.equal(served, y)

    flat = ids.flatten()
    at = 0
    want_gx, bound = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64)
    for e in range(experts):
        choices = (flat == e).nonzero().flatten()
        n = len(choices)
        mine = torch.arange(at, at + n) if sorted_rows else choices // top_k
        x_e, g_e, w_e = x[mine], g[at : at + n], w[e]
        if n:
            assert_product(y[at : at + n], through(x_e), through(w_e))
            assert_product(gw[e], through(g_e.t()), through(x_e.t()))
            gx_e, size = through(g_e) @ through(w_e.t()).t(), through(g_e).abs() @ through(w_e.t()).abs().t()
            want_gx.index_add_(0, mine, gx_e)
            # each choice's part is rounded, then the sum
            bound.index_add_(0, mine, (out_dim + top_k) * 2.0**-23 * size + 2 * ROUNDING[dtype] * (1 + ROUNDING[dtype]) * gx_e.abs())
        else:
            assert not gw[e].any()
        at += n
    assert not y[at:].any()
    if dtype == torch.float16:
        bound += (top_k + 1) * 2.0**-25
    assert ((gx.double().cpu() - want_gx).abs() <= bound + 2.0**-133).all()


@pytest.mark.parametrize(
    "tiles,tokens,top_k,experts,n,k,absent",
    [("64", 30, 2, 9, 300, 700, 0.1), ("128", 900, 4, 30, 2100, 500, 0.0), ("256", 2100, 4, 17, 1290, 600, 0.3)],
)
def test_every_kernel_of_the_experts(device, tiles, tokens, top_k, experts, n, k, absent):
    assert hip_ops.mxfp4_gemm_tiles(tokens * top_k, n, k, mode=_native.MXFP4_ROWS, experts=experts) == tiles
    gen = torch.Generator(device=device).manual_seed(tokens)
    ids = torch.randint(0, experts, (tokens, top_k), generator=gen, device=device)
    ids[: tokens // 3] = experts - 2  # one of them much liked
    ids = torch.where(torch.rand(tokens, top_k, generator=gen, device=device) < absent, -1, ids)
    routing = route_tokens(ids, experts)
    x, w = (torch.randn(*s, generator=gen, device=device) for s in ((tokens, k), (experts, n, k)))
    x.requires_grad_()
    w.requires_grad_()
    g = torch.randn(tokens * top_k, n, generator=gen, device=device)
    y = mxfp4_expert_linear(x, w, routing)
    gx, gw = torch.autograd.grad(y, (x, w), g)

    def on(t):  # the values, in 64 bits
        return mxfp4_quantize(t.detach()).dequantize(torch.float32).double()

    offsets, source = routing.offsets.tolist(), routing.source.long()
    want_gx = torch.zeros(tokens, k, dtype=torch.float64, device=device)
    size_gx = torch.zeros_like(want_gx)
    for e in range(experts):
        part = slice(offsets[e], offsets[e + 1])
        if part.start == part.stop:
            assert not gw[e].any()
            continue
        of = source[part] // top_k
        x_e, w_e, g_e = x[of], w[e], g[part]
        for got, a, b in ((y[part], on(x_e), on(w_e)), (gw[e], on(g_e.t()), on(x_e.t()))):
            want, size = torch.mm(a, b.t()), torch.mm(a.abs(), b.abs().t())
            assert ((got.double() - want).abs() <= a.shape[1] * 2.0**-23 * size + 2.0**-24 * want.abs()).all()
        a, b = on(g_e), on(w_e.t())
        want_gx.index_add_(0, of, torch.mm(a, b.t()))
        size_gx.index_add_(0, of, torch.mm(a.abs(), b.abs().t()))
    assert not y[offsets[-1] :].any()
    assert ((gx.double() - want_gx).abs() <= (n + 2 * top_k) * 2.0**-23 * size_gx).all()


def test_expert_layer_through_the_whole_path(device):
    """Routing, two products with a gate between them and the way back, with
    gradients for everything, against the same layer token by token."""
    tokens, top_k, experts, width, hidden = 50, 2, 6, 96, 64
    x = _normal((tokens, width), 1.0, torch.float32, 1).to(device).requires_grad_()
    up, down = (_normal(s, 0.1, torch.float32, i).to(device).requires_grad_() for i, s in ((2, (experts, hidden, width)), (3, (experts, width, hidden))))
    router = _normal((experts, width), 0.1, torch.float32, 4).to(device).requires_grad_()
    weights, ids = torch.softmax(x @ router.t(), dim=-1).topk(top_k, dim=-1)
    routing = route_tokens(ids, experts)
    h = torch.relu(mxfp4_expert_linear(x, up, routing))
    y = combine_tokens(mxfp4_expert_linear(h, down, routing, sorted_rows=True), routing, weights)
    again = combine_tokens(
        mxfp4_expert_linear(torch.relu(mxfp4_expert_linear(dispatch_tokens(x, routing), up, routing, sorted_rows=True)), down, routing,
                            sorted_rows=True), routing, weights)
    assert torch.equal(y, again)
    want = torch.stack([
        sum(weights[t, j] * mxfp4_linear(torch.relu(mxfp4_linear(x[t : t + 1], up[ids[t, j]])), down[ids[t, j]])[0] for j in range(top_k))
        for t in range(tokens)])
    assert torch.allclose(y, want, rtol=1e-5, atol=1e-6)  # fp32 sums in another order
    grads = torch.autograd.grad(y.square().sum(), (x, up, down, router))
    assert all(torch.isfinite(g).all() and g.any() for g in grads)


def test_graph_replays_and_another_stream(device):
    ids = _ids(40, 2, 6, 5, "few here").to(device)
    x, w = _normal((40, 128), 1.0, torch.bfloat16, 1).to(device), _normal((6, 96, 128), 0.05, torch.bfloat16, 2).to(device)
    dense = quantize_mxfp4_weight(w[0])

    @torch.no_grad()
    def step():
        routing = route_tokens(ids, 6)
        y = mxfp4_expert_linear(x, w, routing)
        return combine_tokens(y, routing, torch.ones(40, 2, device=device)), mxfp4_linear(x, dense)

    want = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        beside = step()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(want, beside))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(_normal((40, 128), 1.0, torch.bfloat16, 10 + i))
        ids.copy_(_ids(40, 2, 6, 20 + i, "few here"))
        for t in out:
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_refusals(device):
    x, w = torch.randn(4, 64, device=device), torch.randn(32, 64, device=device)
    with pytest.raises(ValueError, match="input dim"):
        mxfp4_linear(x[:, :32], w)
    with pytest.raises(NotImplementedError):
        mxfp4_linear(x.double(), w)
    with pytest.raises(NotImplementedError):
        mxfp4_linear(x, w.double())
    with pytest.raises(ValueError, match="bias"):
        mxfp4_linear(x, w, torch.randn(31, device=device))
    with pytest.raises(ValueError, match="weight"):
        mxfp4_linear(x, w[None])
    with pytest.raises(RuntimeError, match="no CPU path"):
        mxfp4_linear(x.cpu(), w.cpu())
    routing = route_tokens(torch.zeros(4, 2, dtype=torch.int64, device=device), 3)
    experts = torch.randn(3, 32, 64, device=device)
    with pytest.raises(ValueError, match="expected weights"):
        mxfp4_expert_linear(x, experts[:2], routing)
    with pytest.raises(ValueError, match="x must be"):
        mxfp4_expert_linear(x, experts, routing, sorted_rows=True)
    with pytest.raises(ValueError, match="x must be"):
        mxfp4_expert_linear(x[:3], experts, routing)
    leaf = x.requires_grad_()
    (first,) = torch.autograd.grad(mxfp4_linear(leaf, w).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), leaf)
