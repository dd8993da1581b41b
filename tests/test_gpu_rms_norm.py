"""Root-mean-square norms and their gradients against the formulas in 64 bits.

Tolerances count roundings, u = 2**-24 each: a row's sum of squares passes at most
60 additions (32 in a thread, the rest between threads), which its root halves; with the
division, the root and the products 64 u are enough for y.  An output rounded to a type of
step eps is off by eps / 2 more."""

import pytest
import torch

from flex_shard_amd import hip_ops
from flex_shard_amd.norms import FlexShardRMSNorm, convert_to_flex_shard_rms_norm, rms_norm, rms_norm_fp8

pytestmark = pytest.mark.gpu

U = 2.0**-24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-5
# types of x and of the residual
PAIRS = [(BF16, None), (BF16, BF16), (BF16, F32), (F16, None), (F16, F16), (F16, F32), (F32, None), (F32, F32)]
# one and more columns, up to the borders of every layout and past them
WIDTHS = [1, 7, 8, 63, 64, 65, 127, 128, 129, 200, 256, 257, 512, 515, 1001, 1024, 2048, 2056, 4095, 4096, 4104, 8192, 8200, 16384, 16385, 20001]


def _step(dtype):
    return torch.finfo(dtype).eps / 2


def _make(rows, cols, dtype, stream, weight=F32, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed + 31 * rows + cols)
    x = (torch.randn(rows, cols, generator=gen, device="cuda") * scale).to(dtype)
    residual = None if stream is None else (2 * torch.randn(rows, cols, generator=gen, device="cuda")).to(stream)
    w = None if weight is None else (1 + 0.3 * torch.randn(cols, generator=gen, device="cuda")).to(weight)
    return x, residual, w, gen


def _norm64(h, w, eps=EPS):
    h = h.double()
    s = 1 / torch.sqrt(h.square().mean(dim=-1, keepdim=True) + eps)
    return h * s * (1 if w is None else w.double()), s


def _check_forward(x, residual, w, eps=EPS):
    with torch.no_grad():
        got = rms_norm(x, w, eps, residual=residual)
    y, total = (got, x) if residual is None else got
    if residual is not None:
        assert total.dtype == residual.dtype
        assert torch.equal(total, (x.float() + residual.float()).to(residual.dtype))
        assert torch.equal(y, rms_norm(x, w, eps, residual=residual)[0])
    assert y.dtype == x.dtype and y.shape == x.shape
    want, _ = _norm64(total, w, eps)
    bound = want.abs() * (_step(x.dtype) + 64 * U) + (2.0**-25 if x.dtype == F16 else 1e-38)
    assert ((y.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("dtype,stream", PAIRS)
def test_widths(dtype, stream, cols):
    x, residual, w, _ = _make(5, cols, dtype, stream)
    _check_forward(x, residual, w)


@pytest.mark.parametrize("cols", [64, 256, 1001, 2048, 4000, 4096, 7168, 8192])
@pytest.mark.parametrize("dtype,stream", PAIRS)
def test_many_rows(dtype, stream, cols):
    """More rows than those that get more lanes each."""
    x, residual, w, _ = _make(777, cols, dtype, stream)
    _check_forward(x, residual, w)


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 63, 1000])
@pytest.mark.parametrize("cols", [64, 130, 700, 2000])
@pytest.mark.parametrize("weight", [None, BF16, F16, F32])
def test_rows_and_weights(rows, cols, weight):
    x, residual, w, _ = _make(rows, cols, BF16, BF16, weight)
    _check_forward(x, residual, w)
    _check_forward(x, None, w)


def test_leading_dimensions_and_strides():
    x, _, w, _ = _make(6, 640, BF16, None)
    want = rms_norm(x, w, EPS)
    assert torch.equal(rms_norm(x.view(2, 3, 640), w, EPS), want.view(2, 3, 640))
    wide = torch.full((6, 1000), 7.0, dtype=BF16, device="cuda")
    for first in (0, 3, 128):  # rows of a wider matrix, at odd addresses too
        wide[:, first : first + 640] = x
        assert torch.equal(rms_norm(wide[:, first : first + 640], w, EPS), want)
    assert torch.equal(rms_norm(x.t().contiguous().t(), w, EPS), want)  # strided columns: copied
    assert torch.equal(rms_norm(x[:1].expand(4, 640), w, EPS), want[:1].expand(4, 640))
    odd = torch.zeros(2 * 640 + 1, dtype=BF16, device="cuda")
    odd[1:] = torch.cat((w.to(BF16), w.to(BF16)))
    assert torch.equal(rms_norm(x, odd[1:641], EPS), rms_norm(x, w.to(BF16), EPS))
    assert torch.equal(rms_norm(x[0], w, EPS), want[0])


def test_one_column_and_zero_rows_of_zeros():
    x = torch.tensor([[3.0], [-2.0], [0.0]], device="cuda")
    assert torch.allclose(rms_norm(x, None, 0.0)[:2], torch.tensor([[1.0], [-1.0]], device="cuda"), rtol=8 * U)
    zeros = torch.zeros(3, 300, dtype=BF16, device="cuda")
    assert torch.equal(rms_norm(zeros, None, EPS), zeros)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_what_is_not_finite_stays_in_its_row(bad):
    x, residual, w, _ = _make(4, 1030, BF16, F32)
    want = rms_norm(x, w, EPS, residual=residual)[0]
    x[2, 77] = bad
    y = rms_norm(x, w, EPS, residual=residual)[0]
    keep = torch.tensor([0, 1, 3], device="cuda")
    assert torch.equal(y[keep], want[keep]) and y[2, 77].isnan()


def test_no_rows():
    x = torch.zeros(0, 64, dtype=BF16, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, total = rms_norm(x, w, residual=torch.zeros(0, 64, device="cuda"))
    assert y.shape == (0, 64) and y.dtype == BF16 and total.dtype == F32
    (y.float().sum() + total.sum()).backward()
    assert torch.equal(w.grad, torch.zeros_like(w)) and x.grad.shape == x.shape


# ---------------------------------------------------------------- gradients
def _grads64(h, w, g, gt, eps=EPS):
    h, g = h.double(), g.double()
    s = 1 / torch.sqrt(h.square().mean(dim=-1, keepdim=True) + eps)
    a, n = g * (1 if w is None else w.double()), h * s
    mean, size = (a * n).mean(dim=-1, keepdim=True), (a * n).abs().mean(dim=-1, keepdim=True)
    dh = s * (a - n * mean) + (0 if gt is None else gt.double())
    # what the roundings are of: both terms, the row's sum of magnitudes, the other gradient
    magnitude = s * (a.abs() + n.abs() * size) + (0 if gt is None else gt.double().abs())
    return dh, magnitude, (g * n).sum(dim=0), (g * n).abs().sum(dim=0)


def _check_grads(x, residual, w, g, gt, got, grad_dtype=None):
    total = x if residual is None else (x.float() + residual.float()).to(residual.dtype)
    dh, magnitude, dw, dw_size = _grads64(total.detach(), w, g, gt)
    outputs = [(got[0], x.dtype)] + ([] if residual is None else [(got[1], residual.dtype)])
    for d, dtype in outputs:
        assert d.dtype == dtype
        # 35 roundings of s, 60 of the sum, and the terms' own
        bound = dh.abs() * _step(dtype) + magnitude * 128 * U + (2.0**-25 if dtype == F16 else 1e-38)
        assert ((d.double() - dh).abs() <= bound).all()
    if w is not None:
        d = got[-1]
        assert d.dtype == w.dtype
        # a column's sum passes fewer additions than there are rows and workgroups' parts
        bound = dw.abs() * _step(w.dtype) + dw_size * (x.shape[0] + 128) * U + (2.0**-25 if w.dtype == F16 else 1e-38)
        assert ((d.double() - dw).abs() <= bound).all()


def _run_grads(x, residual, w, gen, with_total=True):
    leaves = [t.requires_grad_() for t in (x, residual, w) if t is not None]
    y = rms_norm(x, w, EPS, residual=residual)
    outputs = (y,) if residual is None else y
    g = torch.randn(x.shape, generator=gen, device="cuda").to(x.dtype)
    grads = [g]
    if residual is not None:
        grads.append(torch.randn(x.shape, generator=gen, device="cuda").to(residual.dtype) if with_total else None)
    used = [(o, d) for o, d in zip(outputs, grads) if d is not None]
    got = torch.autograd.grad([o for o, _ in used], leaves, [d for _, d in used])
    return g, grads[1] if len(grads) > 1 else None, got


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("dtype,stream", PAIRS)
def test_gradients_of_widths(dtype, stream, cols):
    x, residual, w, gen = _make(5, cols, dtype, stream)
    g, gt, got = _run_grads(x, residual, w, gen)
    _check_grads(x, residual, w, g, gt, got)


@pytest.mark.parametrize("rows,cols", [(1, 64), (17, 130), (3000, 96), (20000, 128), (1100, 600), (1500, 2000), (600, 12000), (515, 17000)])
@pytest.mark.parametrize("weight", [None, BF16, F32])
def test_gradients_of_many_rows(rows, cols, weight):
    for stream, with_total in ((BF16, True), (BF16, False), (F32, True), (None, False)):
        x, residual, w, gen = _make(rows, cols, BF16, stream, weight)
        g, gt, got = _run_grads(x, residual, w, gen, with_total)
        _check_grads(x, residual, w, g, gt, got)


def test_gradients_against_differences():
    x, residual, w, gen = _make(3, 37, F32, F32)
    g, gt, got = _run_grads(x, residual, w, gen)
    for t, d in zip((x, residual, w), got):
        direction = torch.randn(t.shape, generator=gen, device="cuda").double()

        def loss(step):
            moved = [u.detach().double() + (step * direction if u is t else 0) for u in (x, residual, w)]
            total = moved[0] + moved[1]
            return (_norm64(total, moved[2])[0] * g.double()).sum() + (total * gt.double()).sum()

        # the formula's third derivative over 6 times the step squared is far below the step's own rounding
        slope = (loss(1e-4) - loss(-1e-4)) / 2e-4
        assert abs(slope - (d.double() * direction).sum()) <= 1e-5 * (d.double() * direction).abs().sum()


def test_only_what_is_wanted():
    x, residual, w, gen = _make(9, 300, BF16, F32)
    g = torch.randn(9, 300, generator=gen, device="cuda").to(BF16)
    full = _run_grads(x.clone(), residual.clone(), w.clone(), torch.Generator(device="cuda").manual_seed(5))
    for mask in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x.detach(), residual.detach(), w.detach()))]
        y, total = rms_norm(leaves[0], leaves[2], EPS, residual=leaves[1])
        wanted = [t for t in leaves if t.requires_grad]
        for got, want in zip(torch.autograd.grad([y, total], wanted, [full[0], full[1]], allow_unused=True), [d for i, d in enumerate(full[2]) if mask >> i & 1]):
            assert torch.equal(got, want)
    leaf, stream = x.detach().clone().requires_grad_(), residual.detach().clone().requires_grad_()
    _, total = rms_norm(leaf, w.detach(), EPS, residual=stream)
    back = torch.autograd.grad(total, (leaf, stream), full[1])
    assert torch.equal(back[0], full[1].to(BF16)) and torch.equal(back[1], full[1])


def test_gradients_of_strided_rows():
    x, residual, w, gen = _make(20, 200, BF16, BF16)
    want = _run_grads(x.clone(), residual.clone(), w.clone(), torch.Generator(device="cuda").manual_seed(3))
    wide = torch.zeros(20, 500, dtype=BF16, device="cuda")
    wide[:, 11:211], wide[:, 250:450] = x.detach(), residual.detach()
    wide.requires_grad_()
    weight = w.detach().clone().requires_grad_()
    y, total = rms_norm(wide[:, 11:211], weight, EPS, residual=wide[:, 250:450])
    spread = torch.zeros(20, 700, dtype=BF16, device="cuda")
    spread[:, 1:201], spread[:, 401:601] = want[0], want[1]
    dwide, dw = torch.autograd.grad([y, total], (wide, weight), [spread[:, 1:201], spread[:, 401:601]])
    assert torch.equal(dwide[:, 11:211], want[2][0]) and torch.equal(dwide[:, 250:450], want[2][1]) and torch.equal(dw, want[2][2])
    ones = torch.autograd.grad(rms_norm(wide[:, 11:211], weight, EPS).sum(), weight)[0]  # an expanded gradient
    assert torch.isfinite(ones).all()


def test_the_same_bits_every_time():
    x, residual, w, gen = _make(3000, 1000, BF16, BF16)
    runs = [_run_grads(x.clone(), residual.clone(), w.clone(), torch.Generator(device="cuda").manual_seed(9))[2] for _ in range(3)]
    for again in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(again, runs[0]))


def test_the_stream_feeds_the_next_layer():
    """Two layers on one residual stream: the gradients of both norms meet in it."""
    x, residual, w, gen = _make(40, 256, F32, F32)
    parts = [x.requires_grad_(), residual.requires_grad_(), w.requires_grad_()]
    y, total = rms_norm(x, w, EPS, residual=residual)
    z, last = rms_norm(torch.tanh(y), w, EPS, residual=total)
    got = torch.autograd.grad((z.sin() + last).sum(), parts)
    parts64 = [t.detach().double().requires_grad_() for t in parts]
    h = parts64[0] + parts64[1]
    y64 = _norm64(h, parts64[2])[0]
    last64 = h + torch.tanh(y64)
    want = torch.autograd.grad((_norm64(last64, parts64[2])[0].sin() + last64).sum(), parts64)
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= 1e-5 * b.norm()  # some 100 roundings of 2**-24 in every factor


def test_captured_and_replayed():
    x, residual, w, gen = _make(300, 520, BF16, BF16)
    leaves = [t.requires_grad_() for t in (x, residual, w)]
    g = torch.randn(300, 520, generator=gen, device="cuda").to(BF16)

    def once():
        y, total = rms_norm(leaves[0], leaves[2], EPS, residual=leaves[1])
        return [y, total, *torch.autograd.grad([y, total], leaves, [g, g])]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(300, 520, generator=gen, device="cuda").to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        want = once()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_on_another_stream():
    x, residual, w, _ = _make(2000, 4096, BF16, BF16)
    want = rms_norm(x, w, EPS, residual=residual)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        busy = torch.randn(4096, 4096, device="cuda")
        for _ in range(3):
            busy = busy @ busy * 1e-3
        late = x + 0 * busy[0, 0].to(BF16).nan_to_num(0.0, 0.0, 0.0)
        got = rms_norm(late, w, EPS, residual=residual)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_offsets_beyond_32_bits():
    cols, rows = 16384, (1 << 32) // 16384 + 40  # 2**32 elements and some, 8.6 GB
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    x[-40:] = torch.randn(40, cols, device="cuda").to(BF16)
    w = 1 + torch.randn(cols, device="cuda")
    tail = x[-40:].clone().requires_grad_()
    y = rms_norm(x, w, EPS)
    assert torch.equal(y[-40:], rms_norm(tail, w, EPS)) and not y[: rows - 40].any()
    rstd = hip_ops.rms_norm(x, w, EPS, keep_rstd=True)[2]
    g = torch.zeros_like(x)
    g[-40:] = 1
    grads = hip_ops.rms_norm_backward(g, x, w, rstd, BF16)
    del y
    want = torch.autograd.grad(rms_norm(tail, w.requires_grad_(), EPS), (tail, w), torch.ones_like(tail))
    assert torch.equal(grads[0][-40:], want[0])
    assert torch.allclose(grads[2], want[1], rtol=0, atol=200 * U * 40 * 6)  # other orders of 40 terms of up to 6


def test_module_and_conversion():
    model = torch.nn.Sequential(torch.nn.RMSNorm(300, eps=EPS), torch.nn.Sequential(torch.nn.RMSNorm((4, 300)), torch.nn.RMSNorm(8, elementwise_affine=False)))
    model = model.cuda()
    first = model[0].weight
    convert_to_flex_shard_rms_norm(model)
    assert type(model[0]) is FlexShardRMSNorm and model[0].weight is first
    assert type(model[1][0]) is torch.nn.RMSNorm and type(model[1][1]) is FlexShardRMSNorm
    x = torch.randn(5, 300, device="cuda").to(BF16)
    with torch.no_grad():
        assert torch.equal(model[0](x), rms_norm(x, first, EPS))
        y, total = model[0](x, x.float())
        assert torch.equal(y, rms_norm(x, first, EPS, residual=x.float())[0]) and total.dtype == F32
        z = torch.randn(2, 8, device="cuda")
        assert torch.equal(model[1][1](z), rms_norm(z, None, torch.finfo(F32).eps))
    with pytest.raises(ValueError):
        model[0](x[:, :200])


def test_refusals():
    x = torch.randn(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    for call, error in (
        (lambda: rms_norm(x.double()), NotImplementedError),
        (lambda: rms_norm(x, w[:63]), ValueError),
        (lambda: rms_norm(x, w.double()), ValueError),
        (lambda: rms_norm(x, w, -1.0), ValueError),
        (lambda: rms_norm(x, w, float("nan")), ValueError),
        (lambda: rms_norm(x, w, residual=x[:1]), ValueError),
        (lambda: rms_norm(x, w, residual=x.to(BF16)), NotImplementedError),
        (lambda: rms_norm(x[:, :0]), ValueError),
        (lambda: rms_norm(x, w.cpu()), RuntimeError),
        (lambda: hip_ops.rms_norm_backward(x, x, w, w, F32), ValueError),
    ):
        with pytest.raises(error):
            call()
    leaf = x.requires_grad_()
    y = rms_norm(leaf, w)
    (d,) = torch.autograd.grad(y.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), leaf)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
        rms_norm(torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x)), w)


def test_saved_tensors_that_come_back_otherwise():
    """Strided rows that a hook keeps on the host come back contiguous; what stays there is refused."""
    x, residual, w, gen = _make(20, 200, BF16, BF16)
    g = torch.randn(20, 200, generator=gen, device="cuda").to(BF16)
    wide = torch.zeros(20, 500, dtype=BF16, device="cuda")
    wide[:, 11:211] = x.detach()
    rows, weight = wide[:, 11:211].requires_grad_(), w.detach().clone().requires_grad_()
    want = torch.autograd.grad(rms_norm(rows, weight, EPS), (rows, weight), g)
    with torch.autograd.graph.save_on_cpu():
        y = rms_norm(rows, weight, EPS)
    for a, b in zip(torch.autograd.grad(y, (rows, weight), g), want):
        assert torch.equal(a, b)
    for back in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t.flatten()[:-1]):
        with torch.autograd.graph.saved_tensors_hooks(back, lambda t: t):
            y = rms_norm(rows, weight, EPS)
        with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
            torch.autograd.grad(y, (rows, weight), g)


@pytest.mark.parametrize("cols", [*range(1, 34), 393, 771, 1030, 1283, 1539, 1805, 2049, 2305, 3003, 5001, 5119, 6001, 7169, 9001, 12290, 14001])
@pytest.mark.parametrize("dtype,stream", [(BF16, None), (BF16, F32), (F16, F16), (F32, F32)])
def test_row_ends(dtype, stream, cols):
    """Every number of columns behind the last whole vector, in rows with neighbours that are not theirs: no
    value of one row's end counts twice, or gets into another row."""
    rows = 6
    gen = torch.Generator(device="cuda").manual_seed(cols)
    wide = torch.full((rows, cols + 5), float("nan"), device="cuda", dtype=dtype)
    wide[:, 2 : cols + 2] = torch.randn(rows, cols, generator=gen, device="cuda").to(dtype)
    wide[:, cols + 1] *= 3  # the last column weighs the most
    x = wide[:, 2 : cols + 2]
    residual = None if stream is None else torch.randn(rows, cols, generator=gen, device="cuda").to(stream)
    w = (1 + 0.3 * torch.randn(cols, generator=gen, device="cuda")).to(dtype)
    _check_forward(x, residual, w)
    x = x.detach()
    g, gt, got = _run_grads(x, residual, w, gen)
    _check_grads(x, residual, w, g, gt, got)


@pytest.mark.parametrize("cols", [500, 1500, 1777, 2000, 4097, 5120, 6001, 7168])
def test_gradients_of_rows_by_the_thousand(cols):
    """Rows enough that those of 4097 to 7168 columns are dealt out otherwise."""
    for stream in (BF16, F32):
        x, residual, w, gen = _make(2500, cols, BF16, stream, BF16)
        g, gt, got = _run_grads(x, residual, w, gen)
        _check_grads(x, residual, w, g, gt, got)


@pytest.mark.parametrize("scale", [1.0, 0.02, 1e-3])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_a_converted_module_without_eps(dtype, scale):
    """A module that names no eps has that of fp32 whatever the type of its rows, as torch's own: of small bf16 or fp16
    rows another one changes the outputs by a factor."""
    x, _, w, gen = _make(6, 300, dtype, None, weight=dtype, scale=scale)
    g = torch.randn(x.shape, generator=gen, device="cuda").to(dtype)
    model = torch.nn.Sequential(torch.nn.RMSNorm(300, device="cuda", dtype=dtype))
    its = model[0]
    its.weight.data.copy_(w)
    convert_to_flex_shard_rms_norm(model)
    mine = model[0]
    assert type(mine) is FlexShardRMSNorm and mine.eps is None
    rows, others = x.clone().requires_grad_(), x.clone().requires_grad_()
    y, want = mine(rows), _norm64(x, w, torch.finfo(F32).eps)[0]
    least = 2.0**-25 if dtype == F16 else 1e-38
    assert ((y.double() - want).abs() <= want.abs() * (_step(dtype) + 64 * U) + least).all()
    theirs = its(others)  # (which may round the norm before the weight's product too)
    assert theirs.dtype == y.dtype
    assert ((y.double() - theirs.double()).abs() <= want.abs() * (3 * _step(dtype) + 128 * U) + 3 * least).all()
    # gradients, of the formula: dh = s (a - n mean(a n)), each sum's error that of its terms' magnitudes
    got = torch.autograd.grad(y, rows, g)[0].double()
    n, s = _norm64(x, None, torch.finfo(F32).eps)
    a = g.double() * w.double()
    mean, size = (a * n).mean(-1, keepdim=True), (a * n).abs().mean(-1, keepdim=True)
    wanted = s * (a - n * mean)
    assert ((got - wanted).abs() <= wanted.abs() * _step(dtype) + 256 * U * s * (a.abs() + n.abs() * size) + least).all()


def test_a_converted_module_without_eps_in_8_bits():
    x, _, w, _ = _make(6, 300, BF16, None, weight=BF16, scale=0.02)
    model = torch.nn.Sequential(torch.nn.RMSNorm(300, device="cuda", dtype=BF16))
    model[0].weight.data.copy_(w)
    mine = convert_to_flex_shard_rms_norm(model)[0]
    with torch.no_grad():
        got, want = mine(x, fp8=True), rms_norm_fp8(x, w, torch.finfo(F32).eps)
        assert torch.equal(got.q.view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(got.scales, want.scales)
        # an E4M3 value is off by half a step of 2**-3, or of 2**-9 of its scale, which is the largest bf16 value over 448
        values, y = got.dequantize(F32).double(), _norm64(x, w, torch.finfo(F32).eps)[0]
        assert ((values - y).abs() <= y.abs() * (2.0**-4 + 2 * _step(BF16)) + y.abs().amax() * (1 + 2 * _step(BF16)) / 448 * 2.0**-10).all()
