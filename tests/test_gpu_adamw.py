"""AdamW steps of many tensors, the sum of squares that clips them, and the 8-bit
states, against their definitions.

Tolerances count roundings, u = 2**-24.  A clipped gradient has two (the factor's, the
product's); the first moment's term of it two more (1 - b1's own, the product's) and the sum's: 5 u of the
terms' magnitudes.  The second moment's has the two twice, the square's, 1 - b2's, the product's
and the sum's: 2 * 2 + 4 = 8 u.  The quotient of the moments, its factors and its
two roots 24 u of the update; the parameter 3 u and its type's own half step."""

import copy

import pytest
import torch
from adamw_definition import BLOCK, FIRST, SECOND, decode, encode, step64

from flex_shard_amd.adamw import FlexShardAdamW, grad_square_sum

pytestmark = pytest.mark.gpu

U = 2.0**-24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HYPER = dict(lr=2e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
SIZES = [(), (1,), (3,), (127,), (128,), (129,), (1024,), (1025,), (33, 77), (4096,), (0,), (5000,), (2, 3, 501)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _params(shapes, dtype, gen, packed=False):
    """Parameters; packed: back to back in one buffer, at odd addresses."""
    counts = [torch.Size(s).numel() for s in shapes]
    if not packed:
        return [torch.nn.Parameter(torch.randn(s, generator=gen, device="cuda").to(dtype)) for s in shapes]
    flat = torch.randn(sum(counts) + 1, generator=gen, device="cuda").to(dtype)
    starts = [1 + sum(counts[:i]) for i in range(len(counts))]
    return [torch.nn.Parameter(flat[a : a + n].view(s)) for a, n, s in zip(starts, counts, shapes)]


def _set_grads(params, dtype, gen, scale=1e-2):
    for p in params:
        p.grad_dtype = None
        p.grad = (torch.randn(p.shape, generator=gen, device="cuda") * scale).to(dtype)


def _check_step(optimizer, params, t, clip=1.0, hyper=HYPER, **arguments):
    before = []
    for p in params:
        m, v = optimizer.state_values(p) if optimizer.state.get(p) else (torch.zeros(p.shape, device="cuda"),) * 2
        before.append((p.detach().clone(), p.grad.clone(), m.clone(), v.clone()))
    optimizer.step(**arguments)
    for p, (p0, g, m0, v0) in zip(params, before):
        want = step64(p0, g, m0, v0, t, clip=clip, **hyper)
        state = optimizer.state[p]
        assert int(state["step"]) == t
        b1, b2 = hyper["betas"]
        g = g.double() * clip
        m_bound = 5 * U * (b1 * m0.abs() + (1 - b1) * g.abs()) + 1e-44
        v_bound = 8 * U * want[2] + 1e-44
        if state["exp_avg"].dtype == F32:
            assert ((state["exp_avg"].double() - want[1]).abs() <= m_bound).all()
            assert ((state["exp_avg_sq"].double() - want[2]).abs() <= v_bound).all()
        update = want[0] - p0.double() * (1 - hyper["lr"] * hyper["weight_decay"])
        # (the first moment's rounding is of its terms, which may cancel)
        relative = torch.where(want[1] == 0, 0.0, m_bound / want[1].abs().clamp(min=1e-44))
        bound = update.abs() * (24 * U + relative) + p0.double().abs() * 3 * U + want[0].abs() * (torch.finfo(p.dtype).eps / 2 if p.dtype != F32 else U)
        assert ((p.detach().double() - want[0]).abs() <= bound + 1e-38).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("grad_dtype", [BF16, F32])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_steps(dtype, grad_dtype, packed, bits):
    gen = _gen(1)
    params = _params(SIZES, dtype, gen, packed)
    optimizer = FlexShardAdamW(params, **HYPER, state_bits=bits)
    for t in range(1, 5):
        _set_grads(params, grad_dtype, gen)
        _check_step(optimizer, params, t)


def test_neighbours_are_left_alone():
    gen = _gen(2)
    flat = torch.full((10000,), 7.0, device="cuda")
    params = [torch.nn.Parameter(flat[a : a + n]) for a, n in ((5, 1), (10, 130), (201, 1023), (2000, 4097))]
    for bits in (32, 8):
        optimizer = FlexShardAdamW(params, **HYPER, state_bits=bits)
        _set_grads(params, F32, gen)
        optimizer.step()
    touched = torch.zeros(10000, dtype=torch.bool, device="cuda")
    for a, n in ((5, 1), (10, 130), (201, 1023), (2000, 4097)):
        touched[a : a + n] = True
    assert (flat[~touched] == 7).all() and (flat[touched] != 7).all()


# ------------------------------------------------------------------ 8-bit states
def _exact_fp32_moments(p0, g, m, v, betas):
    """The moments in the kernel's own order of fp32 operations."""
    b1, b2 = betas
    g = g.float()
    return m * b1 + g * (1 - b1), v * b2 + (g * g) * (1 - b2)


@pytest.mark.parametrize("n", [1, 100, 128, 130, 5000, 70001])
@pytest.mark.parametrize("spread", [1.0, 30.0])
def test_codes_are_the_definitions(n, spread):
    """Bit for bit, over magnitudes from a block's largest to far below its smallest code."""
    gen = _gen(n)
    p = torch.nn.Parameter(torch.randn(n, generator=gen, device="cuda"))
    optimizer = FlexShardAdamW([p], **HYPER, state_bits=8)
    m = v = torch.zeros(n)
    for t in range(1, 6):
        p.grad = torch.randn(n, generator=gen, device="cuda") * torch.exp(-spread * torch.rand(n, generator=gen, device="cuda"))
        p.grad[torch.rand(n, generator=gen, device="cuda") < 0.1] = 0
        optimizer.step()
        m, v = _exact_fp32_moments(None, p.grad.cpu(), m, v, HYPER["betas"])
        state = optimizer.state[p]
        for name, value, which in (("exp_avg", m, FIRST), ("exp_avg_sq", v, SECOND)):
            code, scale = encode(value, t, which)
            assert torch.equal(state[name].cpu(), code) and torch.equal(state[f"{name}_scale"].cpu(), scale), (name, t)
        m = decode(state["exp_avg"].cpu(), state["exp_avg_scale"].cpu(), FIRST)
        v = decode(state["exp_avg_sq"].cpu(), state["exp_avg_sq_scale"].cpu(), SECOND)
        for dtype in (F32, BF16, F16):
            got = optimizer.state_values(p, dtype)
            assert torch.equal(got[0].cpu(), m.to(dtype)) and torch.equal(got[1].cpu(), v.to(dtype))


def test_second_moment_moves_at_its_rate():
    """With gradients of zero the second moment has to fall by 1 - b2 a step, which
    is less than half a code's step: rounded to nearest it would stay."""
    n, b2, steps = 128 * 200, 0.99, 300
    gen = _gen(3)
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    optimizer = FlexShardAdamW([p], lr=0.0, betas=(0.9, b2), weight_decay=0.0, state_bits=8)
    p.grad = torch.rand(n, generator=gen, device="cuda") + 0.1
    p.grad[::BLOCK] = 2.0
    optimizer.step()
    first = optimizer.state_values(p)[1].double()
    # (a block's largest has the scale, which follows it exactly: gradients that keep it let the others fall)
    p.grad = torch.zeros(n, device="cuda")
    p.grad[::BLOCK] = (optimizer.state_values(p)[1][::BLOCK]).sqrt()
    for _ in range(steps):
        optimizer.step()
    last = optimizer.state_values(p)[1].double()
    others = torch.arange(n, device="cuda") % BLOCK != 0
    ratio = (last[others].mean() / first[others].mean()).item()
    # a walk of 300 steps of an eighth of an octave, averaged over 25400 elements, is within a few per cent
    assert abs(ratio / b2**steps - 1) < 0.1


def test_not_finite_blocks():
    p = torch.nn.Parameter(torch.ones(512, device="cuda"))
    optimizer = FlexShardAdamW([p], **HYPER, state_bits=8)
    p.grad = torch.ones(512, device="cuda")
    p.grad[130] = float("nan")
    p.grad[400] = float("inf")
    optimizer.step()
    assert p[:128].isfinite().all() and p[256:384].isfinite().all() and p[130].isnan()
    m, v = optimizer.state_values(p)
    for values in (m, v):
        assert values[:128].isfinite().all() and values[256:384].isfinite().all()
        assert values[128:256].isnan().all() and values[384:].isnan().all()


# --------------------------------------------------------- clipping, what it skips
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_clipped(max_norm, bits):
    gen = _gen(4)
    params = _params(SIZES, F32, gen)
    optimizer = FlexShardAdamW(params, **HYPER, state_bits=bits)
    for t in range(1, 4):
        _set_grads(params, F32, gen, 0.1)
        square_sum = grad_square_sum([p.grad for p in params])
        norm = sum(p.grad.double().square().sum() for p in params).sqrt()
        _check_step(optimizer, params, t, min(1.0, max_norm / (norm.item() + 1e-6)), square_sum=square_sum, max_norm=max_norm)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_sum_that_is_not_finite_skips_the_step(bad, bits):
    gen = _gen(5)
    params = _params([(300,), (1000,)], BF16, gen)
    optimizer = FlexShardAdamW(params, **HYPER, state_bits=bits)
    _set_grads(params, BF16, gen)
    optimizer.step()
    before = copy.deepcopy((params, optimizer.state_dict()["state"]))
    params[1].grad[3] = bad
    optimizer.step(square_sum=grad_square_sum([p.grad for p in params]), max_norm=1.0)
    after = (params, optimizer.state_dict()["state"])
    assert all(torch.equal(a, b) for a, b in zip(before[0], after[0]))
    for i, state in before[1].items():
        assert all(torch.equal(value, after[1][i][name]) for name, value in state.items())
    optimizer.step(square_sum=torch.tensor(bad, dtype=torch.float64, device="cuda"))  # without clipping too
    assert all(torch.equal(a, b) for a, b in zip(before[0], params))
    params[1].grad[3] = 0
    optimizer.step(square_sum=grad_square_sum([p.grad for p in params]), max_norm=1.0)
    assert int(optimizer.state[params[0]]["step"]) == 2 and not torch.equal(before[0][0], params[0])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("sizes", [[1], [7, 0, 8191, 8192, 8193], [3] * 32, [8192] * 31 + [0, 9], [3] * 33, [3] * 400, [1 << 20, 5], [25_000_003], [140_000_000, 77]])
def test_square_sums(sizes, dtype):
    gen = _gen(6)
    flat = torch.randn(sum(sizes) + 1, generator=gen, device="cuda").to(dtype)
    parts = list(flat[1:].split(sizes))
    got = grad_square_sum([None, *parts])
    want = sum(p.double().square().sum() for p in parts)
    # squares of at most 24 bits are exact in 53; the sums' roundings, at most one for each of 4096 in a row
    assert got.dtype == torch.float64 and got.shape == () and abs(got - want) <= 2 * 4096 * 2.0**-53 * want
    assert torch.equal(got, grad_square_sum(parts))


def test_square_sums_of_extremes():
    large = torch.full((1000,), 3e38, device="cuda")
    want = 1000 * (large[0].double() ** 2)
    assert abs(grad_square_sum([large]) / want - 1) < 1e-12
    mixed = [torch.ones(5, device="cuda", dtype=d) for d in (BF16, F16, F32)]
    assert grad_square_sum(mixed).item() == 15
    assert grad_square_sum([torch.arange(12, device="cuda", dtype=F32).view(3, 4).t()]).item() == 506
    assert grad_square_sum([torch.zeros(0, device="cuda")]).item() == 0


# ------------------------------------------------------------------- the optimizer
def test_groups_and_missing_gradients():
    gen = _gen(7)
    params = _params([(500,)] * 40, F32, gen)
    hypers = [dict(lr=1e-3 * (i + 1), betas=(0.8 + 0.005 * i, 0.9), eps=1e-7, weight_decay=0.01 * i) for i in range(20)]
    optimizer = FlexShardAdamW([dict(params=params[2 * i : 2 * i + 2], **h) for i, h in enumerate(hypers)])
    counts = [0] * 40
    for round_ in range(3):
        _set_grads(params, F32, gen)
        for i in range(0, 40, 7):
            if round_ != 1:
                params[i].grad = None
        before = [p.detach().clone() for p in params]
        states = [tuple(s.clone() for s in optimizer.state_values(p)) if optimizer.state.get(p) else (torch.zeros(500, device="cuda"),) * 2 for p in params]
        optimizer.step()
        for i, p in enumerate(params):
            if p.grad is None:
                assert torch.equal(p, before[i])
                continue
            counts[i] += 1
            want = step64(before[i], p.grad, *states[i], counts[i], **hypers[i // 2])[0]
            assert torch.allclose(p.detach().double(), want, rtol=8 * U, atol=1e-8)
            assert int(optimizer.state[p]["step"]) == counts[i]


def test_follows_torchs_own():
    gen = _gen(8)
    params = _params([(64, 64), (1000,)], F32, gen)
    others = [torch.nn.Parameter(p.detach().clone()) for p in params]
    mine, its = FlexShardAdamW(params, **HYPER), torch.optim.AdamW(others, **HYPER)
    schedule = [torch.optim.lr_scheduler.LinearLR(o, 0.1, 1.0, 10) for o in (mine, its)]
    for _ in range(10):
        _set_grads(params, F32, gen)
        for p, q in zip(params, others):
            q.grad = p.grad.clone()
        for optimizer, scheduler in zip((mine, its), schedule):
            optimizer.step()
            scheduler.step()
    for p, q in zip(params, others):
        # ten updates of at most some lr, each with some 30 roundings
        assert (p - q).abs().max() <= 10 * (HYPER["lr"] * 5 * 60 * U + 4 * U * p.abs().max())
    resumed = FlexShardAdamW([torch.nn.Parameter(q.detach().clone()) for q in others], **HYPER)
    saved = its.state_dict()
    for group in saved["param_groups"]:
        group["state_bits"] = 32
    resumed.load_state_dict(saved)
    for p, q in zip(resumed.param_groups[0]["params"], others):
        assert torch.equal(resumed.state[p]["exp_avg"], its.state[q]["exp_avg"]) and int(resumed.state[p]["step"]) == 10


@pytest.mark.parametrize("bits", [32, 8])
def test_saved_and_resumed(bits, tmp_path):
    gen = _gen(9)
    params = _params(SIZES, BF16, gen)
    optimizer = FlexShardAdamW(params, **HYPER, state_bits=bits)
    for _ in range(2):
        _set_grads(params, BF16, gen)
        optimizer.step()
    torch.save(optimizer.state_dict(), tmp_path / "state.pt")
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    resumed = FlexShardAdamW(twins, **HYPER, state_bits=bits)
    resumed.load_state_dict(torch.load(tmp_path / "state.pt", weights_only=True))
    for _ in range(2):
        _set_grads(params, BF16, gen)
        for p, q in zip(params, twins):
            q.grad = p.grad.clone()
        optimizer.step()
        resumed.step()
    for p, q in zip(params, twins):
        assert torch.equal(p, q)
        for name, value in optimizer.state[p].items():
            assert torch.equal(value, resumed.state[q][name]) and value.dtype == resumed.state[q][name].dtype
    other = FlexShardAdamW(twins, **HYPER, state_bits=40 - bits)
    bad = optimizer.state_dict()
    bad["param_groups"][0]["state_bits"] = 40 - bits
    with pytest.raises(ValueError, match="states need"):
        other.load_state_dict(bad)


def test_bits_do_not_depend_on_the_company():
    """A tensor's step is the same alone, among many, and on every run."""
    gen = _gen(10)
    shapes = [(1000 + i,) for i in range(150)]
    params = _params(shapes, BF16, gen)
    alone = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for bits in (32, 8):
        together = FlexShardAdamW(params, **HYPER, state_bits=bits)
        singles = [FlexShardAdamW([p], **HYPER, state_bits=bits) for p in alone]
        for _ in range(2):
            _set_grads(params, BF16, gen)
            for p, q in zip(params, alone):
                q.grad = p.grad.clone()
            together.step()
            for optimizer in singles:
                optimizer.step()
        assert all(torch.equal(p, q) for p, q in zip(params, alone))


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(bits):
    gen = _gen(11)
    params = _params([(4000,), (129,)], F32, gen)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    _set_grads(params, F32, gen)
    _set_grads(twins, F32, gen)
    lr = torch.tensor(1e-3, device="cuda")
    captured = FlexShardAdamW(params, lr=lr, state_bits=bits)
    eager = FlexShardAdamW(twins, lr=lr.item(), state_bits=bits)  # (the same number: fp32 has no 1e-3)
    for _ in range(1):  # the states must exist
        for p, q in zip(params, twins):
            q.grad.copy_(p.grad)
        captured.step(square_sum=grad_square_sum([p.grad for p in params]), max_norm=0.1)
        eager.step(square_sum=grad_square_sum([p.grad for p in twins]), max_norm=0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step(square_sum=grad_square_sum([p.grad for p in params]), max_norm=0.1)
    for i in range(4):
        rate = 1e-3 * (i + 1)
        lr.fill_(rate)
        eager.param_groups[0]["lr"] = float(torch.tensor(rate))
        for p, q in zip(params, twins):
            p.grad.copy_(torch.randn(p.shape, generator=gen, device="cuda"))
            q.grad.copy_(p.grad)
        if i == 2:  # a step that is skipped
            params[0].grad[5] = twins[0].grad[5] = float("inf")
        graph.replay()
        eager.step(square_sum=grad_square_sum([p.grad for p in twins]), max_norm=0.1)
        torch.cuda.synchronize()
        for p, q in zip(params, twins):
            assert torch.equal(p, q)
            assert all(torch.equal(value, eager.state[q][name]) for name, value in captured.state[p].items())
    assert int(captured.state[params[0]]["step"]) == 4


def test_states_are_not_made_in_a_capture():
    p = torch.nn.Parameter(torch.zeros(10, device="cuda"))
    p.grad = torch.ones(10, device="cuda")
    optimizer = FlexShardAdamW([p])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before it is captured"):
        with torch.cuda.graph(graph):
            optimizer.step()


def test_on_another_stream():
    gen = _gen(12)
    params = _params([(3_000_000,), (77,)], F32, gen)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    mine, other = FlexShardAdamW(params, **HYPER), FlexShardAdamW(twins, **HYPER)
    _set_grads(params, F32, gen)
    for p, q in zip(params, twins):
        q.grad = torch.zeros_like(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        busy = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            busy = busy @ busy * 1e-3
        for p, q in zip(params, twins):
            q.grad.copy_(p.grad)
        other.step(square_sum=grad_square_sum([q.grad for q in twins]), max_norm=1.0)
    mine.step(square_sum=grad_square_sum([p.grad for p in params]), max_norm=1.0)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(params, twins))


def test_versions_and_closures():
    p = torch.nn.Parameter(torch.randn(10, device="cuda"))
    optimizer = FlexShardAdamW([p])

    def closure():
        optimizer.zero_grad()
        loss = p.square().sum()
        loss.backward()
        return loss

    assert optimizer.step(closure).item() > 0
    kept = (p * p).sum()
    p.grad = torch.ones_like(p)
    optimizer.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()


def test_offsets_beyond_32_bits():
    n = (1 << 32) + 1000
    p = torch.nn.Parameter(torch.zeros(n, dtype=BF16, device="cuda"))
    p.grad = torch.zeros(n, dtype=BF16, device="cuda")
    gen = _gen(13)
    tail = (torch.randn(1000, generator=gen, device="cuda")).to(BF16)
    p.grad[-1000:] = tail
    with torch.no_grad():
        p[-1000:] = 1
    # blocks begin at multiples of 128: 2**32 is one, so the last 1000 are a tensor's first ones
    q = torch.nn.Parameter(torch.ones(1000, dtype=BF16, device="cuda"))
    q.grad = tail.clone()
    big, small = (FlexShardAdamW([t], **HYPER, state_bits=8) for t in (p, q))
    for _ in range(2):
        square_sum = grad_square_sum([p.grad])
        want = tail.double().square().sum()
        assert abs(square_sum - want) <= 1e-12 * want
        big.step(square_sum=square_sum, max_norm=1.0)
        small.step(square_sum=grad_square_sum([q.grad]), max_norm=1.0)
    assert torch.equal(p[-1000:], q) and not p[:-1000].any()
    for name in ("exp_avg", "exp_avg_sq"):
        assert torch.equal(big.state[p][name][-1000:], small.state[q][name])
        assert torch.equal(big.state[p][f"{name}_scale"][-8:], small.state[q][f"{name}_scale"])


def test_refusals():
    p = torch.nn.Parameter(torch.zeros(16, device="cuda"))
    p.grad = torch.ones(16, device="cuda")
    for arguments, error in (
        (dict(betas=(1.0, 0.9)), ValueError), (dict(betas=(0.9, -0.1)), ValueError), (dict(eps=-1.0), ValueError),
        (dict(weight_decay=-1.0), ValueError), (dict(lr=-1.0), ValueError), (dict(state_bits=4), NotImplementedError),
    ):
        with pytest.raises(error):
            FlexShardAdamW([p], **arguments)
    with pytest.raises(NotImplementedError):
        FlexShardAdamW([torch.nn.Parameter(torch.zeros(4, device="cuda", dtype=F16))])
    optimizer = FlexShardAdamW([p])
    with pytest.raises(ValueError, match="max_norm"):
        optimizer.step(max_norm=1.0)
    with pytest.raises(ValueError, match="max_norm"):
        optimizer.step(square_sum=grad_square_sum([p.grad]), max_norm=0.0)
    with pytest.raises(ValueError, match="float64"):
        optimizer.step(square_sum=torch.ones((), device="cuda"))
    with pytest.raises(ValueError, match="float64 on cuda"):
        optimizer.step(square_sum=torch.ones((), dtype=torch.float64))
    q = torch.nn.Parameter(torch.zeros(4, 4, device="cuda").t()[:, :3])
    q.grad = torch.zeros(4, 3, device="cuda")
    with pytest.raises(ValueError, match="contiguous"):
        FlexShardAdamW([q]).step()
    p.grad_dtype = None
    p.grad = torch.ones(16, device="cuda", dtype=F16)
    with pytest.raises(NotImplementedError):
        optimizer.step()
    assert not p.any()
    with pytest.raises(ValueError):
        grad_square_sum([None])
    with pytest.raises(NotImplementedError):
        grad_square_sum([torch.zeros(3, device="cuda", dtype=torch.float64)])
    with pytest.raises(RuntimeError):
        grad_square_sum([torch.zeros(3)])
    with pytest.raises(KeyError):
        optimizer.state_values(p)


@pytest.mark.parametrize("bits", [32, 8])
def test_replaced_states_and_parameters_listed_twice(bits):
    p = torch.nn.Parameter(torch.zeros(300, device="cuda"))
    p.grad = torch.ones(300, device="cuda")
    optimizer = FlexShardAdamW([p], state_bits=bits)
    optimizer.step()
    before = p.detach().clone()
    state = dict(optimizer.state[p])
    for name, kept in state.items():
        for other in (kept.double(), kept.cpu(), kept.reshape(-1)[:0]):
            optimizer.state[p][name] = other
            with pytest.raises(ValueError, match=name):
                optimizer.step()
        optimizer.state[p][name] = kept
    p.data = torch.zeros(400, device="cuda")  # a parameter that has grown
    p.grad = torch.ones(400, device="cuda")
    with pytest.raises(ValueError, match="exp_avg"):
        optimizer.step()
    whole = torch.zeros(300, device="cuda")
    parts = [torch.nn.Parameter(whole), torch.nn.Parameter(whole[100:200])]
    for t in parts:
        t.grad = torch.ones_like(t)
    with pytest.raises(RuntimeError, match="overlap"):
        FlexShardAdamW(parts, state_bits=bits).step()
    assert before.any() and not p.any() and not whole.any()
    values = optimizer.state_values(p)
    values[0].zero_()  # (a copy)
    assert optimizer.state_values(p)[0].any()


def test_more_tensors_than_a_table_holds():
    """300 tensors: two launches of the factors, five of the steps, two of the sums."""
    gen = _gen(21)
    params = _params([(40 + i,) for i in range(300)], F32, gen)
    _set_grads(params, BF16, gen)
    total = grad_square_sum([p.grad for p in params])
    want = sum(p.grad.double().square().sum() for p in params)
    assert abs(total / want - 1) < 1e-12  # (sums of some 57000 squares in 64 bits)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for p, q in zip(params, twins):
        q.grad_dtype = None  # (any type)
        q.grad = p.grad.clone()
    optimizer = FlexShardAdamW(params, **HYPER)
    optimizer.step(square_sum=total, max_norm=0.5)
    for q in twins:
        FlexShardAdamW([q], **HYPER).step(square_sum=total, max_norm=0.5)
    assert all(torch.equal(p, q) for p, q in zip(params, twins))
    assert all(int(optimizer.state[p]["step"]) == 1 for p in params)


@pytest.mark.parametrize("sizes", [[131072], [131073], [8192] * 16, [8192] * 15 + [8191, 2], [65536, 0, 65536], [4096] * 31 + [1]])
def test_square_sums_around_a_single_workgroups_share(sizes):
    gen = _gen(22)
    for dtype in (BF16, F32):
        parts = [torch.randn(n, generator=gen, device="cuda").to(dtype) for n in sizes]
        want = sum(p.double().square().sum() for p in parts)
        assert abs(grad_square_sum(parts) - want) <= 2 * 4096 * 2.0**-53 * want


def _learning_rates(captured):
    """A step of two groups, the first without gradients, with one learning rate on the GPU, and its twin's with a number."""
    gen = _gen(23)
    params = _params([(300,), (300,)], F32, gen)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    lr = torch.tensor(2e-3, device="cuda")
    mine = FlexShardAdamW([dict(params=[p]) for p in params], lr=lr)
    other = FlexShardAdamW([dict(params=[q]) for q in twins], lr=lr.item())
    _set_grads(params[1:], F32, gen)
    twins[1].grad = params[1].grad.clone()
    other.step()
    if captured:
        mine.step()  # the states must exist
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            mine.step()
        for _ in range(3):
            graph.replay()
            other.step()
            torch.cuda.synchronize()
            assert torch.equal(params[1], twins[1])
    else:
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("error")
        try:
            mine.step()
        finally:
            torch.cuda.set_sync_debug_mode("default")
    assert torch.equal(params[1], twins[1]) and torch.equal(params[0], twins[0])
    assert not mine.state.get(params[0])


def test_learning_rate_on_the_gpu_of_a_group_without_gradients():
    """Nothing waits for the GPU."""
    _learning_rates(captured=False)


def test_learning_rate_on_the_gpu_of_a_group_without_gradients_captured():
    _learning_rates(captured=True)


@pytest.mark.parametrize("bits", [32, 8])
def test_nothing_is_stepped_when_a_late_group_is_refused(bits):
    """More groups than one launch takes: all are checked before the first is stepped."""
    gen = _gen(24)
    params = _params([(200,)] * 20, F32, gen)
    whole = torch.zeros(300, device="cuda")
    params[1], params[18] = (torch.nn.Parameter(whole[a : a + 200]) for a in (0, 100))
    _set_grads(params, F32, gen)
    before = [p.detach().clone() for p in params]
    versions = [p._version for p in params]
    optimizer = FlexShardAdamW([dict(params=[p]) for p in params], **HYPER, state_bits=bits)
    with pytest.raises(RuntimeError, match="overlap"):
        optimizer.step()
    params[18].data = torch.zeros(200, device="cuda")
    optimizer.param_groups[19]["betas"] = (0.9, 1.0)
    with pytest.raises(RuntimeError, match="betas"):
        optimizer.step()
    before[18].zero_()
    assert all(torch.equal(p, q) for p, q in zip(params, before)) and versions == [p._version for p in params]
    assert all(int(optimizer.state[p]["step"]) == 0 for p in params)
    optimizer.param_groups[19]["betas"] = HYPER["betas"]
    optimizer.step()
    assert all(int(optimizer.state[p]["step"]) == 1 for p in params)
    for p, q in zip(params, before):
        want = step64(q, p.grad, torch.zeros_like(q), torch.zeros_like(q), 1, **HYPER)[0]
        assert torch.allclose(p.detach().double(), want, rtol=8 * U, atol=1e-8)
