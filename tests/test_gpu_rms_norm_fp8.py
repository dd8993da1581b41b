"""The norm in 8 bits: the bits of the norm in bf16 behind the linears' quantizer,
and the linears that take it."""

import pytest
import torch

from flex_shard_amd import hip_ops
from flex_shard_amd.blockwise_fp8 import (
    BlockwiseFp8Weight, Fp8Activation, FlexShardFloat8BlockwiseLinear, prequantized_linear,
)
from flex_shard_amd.norms import FlexShardRMSNorm, rms_norm, rms_norm_fp8

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6
# types of which the bf16 norm can be had elsewhere in the same bits: fp32 and bf16
PAIRS = [(BF16, None), (BF16, BF16), (BF16, F32), (F32, None), (F32, F32)]
WIDTHS = [1, 8, 64, 100, 128, 130, 256, 257, 520, 1000, 1024, 2048, 2050, 4096, 4232, 7168, 8192, 8200, 12288, 16384, 16390, 20001]


def _make(rows, cols, dtype, stream, weight=F32):
    gen = torch.Generator(device="cuda").manual_seed(rows * 7919 + cols)
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x[:, ::37] *= 20
    residual = None if stream is None else torch.randn(rows, cols, generator=gen, device="cuda").to(stream)
    w = None if weight is None else (1 + 0.3 * torch.randn(cols, generator=gen, device="cuda")).to(weight)
    return x.to(dtype), residual, w, gen


def _quantized(y):
    """The quantizer's bytes and scales of y in bf16, columns padded to what it reads."""
    y = y.to(BF16)
    return torch.nn.functional.pad(y, (0, -y.shape[1] % 8)).contiguous()


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("dtype,stream", PAIRS)
def test_bits_of_the_norm_and_the_quantizer(dtype, stream, cols):
    x, residual, w, _ = _make(37, cols, dtype, stream)
    if dtype == BF16 and cols % 5 == 0:
        w = None
    got, want = rms_norm_fp8(x, w, EPS, residual=residual), rms_norm(x, w, EPS, residual=residual)
    if residual is not None:
        (got, total), (want, total2) = got, want
        assert torch.equal(total, total2)
    padded = _quantized(want)
    q, scales = hip_ops.act_quant_1x128(padded)
    assert isinstance(got, Fp8Activation) and got.shape == x.shape
    assert _same(got.q, q) and torch.equal(got.scales, scales)
    runs, runs_scales = hip_ops.act_quant_128x1_transposed(padded)
    mine, mine_scales = got.token_runs()
    assert _same(mine, runs) and torch.equal(mine_scales, runs_scales)
    assert got.token_runs()[0] is mine


@pytest.mark.parametrize("cols", [64, 700, 2048, 4096, 7168])
@pytest.mark.parametrize("rows", [1, 5, 16, 127, 128, 129, 300, 600])
def test_rows(rows, cols):
    x, residual, w, _ = _make(rows, cols, BF16, BF16, BF16)
    got, _ = rms_norm_fp8(x, w, EPS, residual=residual)
    padded = _quantized(rms_norm(x, w, EPS, residual=residual)[0])
    assert _same(got.q, hip_ops.act_quant_1x128(padded)[0])
    assert _same(got.token_runs()[0], hip_ops.act_quant_128x1_transposed(padded)[0])


@pytest.mark.parametrize("stream", [None, F16, F32])
def test_fp16_rows(stream):
    """No other call has the bf16 norm of fp16 rows in the same bits: the values are
    within an E4M3 rounding, a bf16 one, and the scale's."""
    x, residual, w, _ = _make(50, 1000, F16, stream)
    got = rms_norm_fp8(x, w, EPS, residual=residual)
    got = got if residual is None else got[0]
    h = x.double() if residual is None else (x.float() + residual.float()).to(residual.dtype).double()
    want = h / torch.sqrt(h.square().mean(dim=1, keepdim=True) + EPS) * w.double()
    runs = torch.nn.functional.pad(want, (0, 24)).view(50, 8, 128)
    least = runs.abs().amax(dim=2, keepdim=True) / 448 * 2.0**-10  # half the smallest step
    bound = (runs.abs() * (2.0**-4 + 2.0**-8 + 2.0**-18) + least * 1.01).view(50, 1024)[:, :1000]
    assert ((got.dequantize(F32).double() - want).abs() <= bound).all()


def test_values():
    x, _, w, _ = _make(33, 300, BF16, None)
    a = rms_norm_fp8(x.view(3, 11, 300), w, EPS)
    q = a.q.float().view(33, 3, 128) * a.scales.t()[:, :, None]
    want = q.view(33, 384)[:, :300].view(3, 11, 300)
    for dtype in (F32, BF16, F16):
        assert torch.equal(a.dequantize(dtype), want.to(dtype))


def test_zeros_and_not_finite():
    x = torch.zeros(4, 256, dtype=BF16, device="cuda")
    a = rms_norm_fp8(x, None, EPS)
    assert not a.dequantize().any() and torch.isfinite(a.scales).all()
    x[1, 3] = float("nan")
    padded = _quantized(rms_norm(x, None, EPS))
    a = rms_norm_fp8(x, None, EPS)
    assert _same(a.q, hip_ops.act_quant_1x128(padded)[0])


# ------------------------------------------------------------------ the linears
def _weight(n, k, gen, requires_grad=True):
    q = (torch.randn(n, k, generator=gen, device="cuda") * 100).clamp(-448, 448).to(torch.float8_e4m3fn)  # (torch's cast of more is a NaN)
    scales = 2e-4 * (1 + torch.rand(-(-n // 128), -(-k // 128), generator=gen, device="cuda"))
    return BlockwiseFp8Weight(q, scales, 128, BF16, requires_grad)


@pytest.mark.parametrize("k", [256, 1000, 130])
@pytest.mark.parametrize("shape", [(70,), (2, 35), (1,)])
def test_linears_take_it(k, shape):
    """The same bits as with the bf16 norm, forward and backward, for two linears
    on one norm."""
    gen = torch.Generator(device="cuda").manual_seed(k)
    weights = [_weight(192, k, gen), _weight(136, k, gen)]
    bias = torch.randn(192, generator=gen, device="cuda").to(BF16).requires_grad_()
    x, residual = (torch.randn(*shape, k, generator=gen, device="cuda").to(BF16).requires_grad_() for _ in range(2))
    norm_weight = (1 + 0.2 * torch.randn(k, generator=gen, device="cuda")).requires_grad_()
    grads = [torch.randn(*shape, n, generator=gen, device="cuda").to(BF16) for n in (192, 136)]
    grad_total = torch.randn(*shape, k, generator=gen, device="cuda").to(BF16)

    def once(norm):
        a, total = norm(x, norm_weight, EPS, residual=residual)
        outs = [prequantized_linear(a, weights[0], bias), prequantized_linear(a, weights[1])]
        leaves = [x, residual, norm_weight, bias, *weights]
        return [*outs, total, *torch.autograd.grad([*outs, total], leaves, [*grads, grad_total])]

    wanted = once(rms_norm)
    for got, want in zip(once(rms_norm_fp8), wanted):
        assert got.shape == want.shape and got.dtype == want.dtype and _same(got.detach(), want.detach())
    with torch.no_grad():
        a, _ = rms_norm_fp8(x, norm_weight, EPS, residual=residual)
        assert _same(prequantized_linear(a, weights[0], bias), wanted[0].detach())


def test_frozen_linear_and_dequantized_gradient():
    gen = torch.Generator(device="cuda").manual_seed(1)
    weight = _weight(128, 256, gen, requires_grad=False)
    x = torch.randn(20, 256, generator=gen, device="cuda").to(BF16).requires_grad_()
    g = torch.randn(20, 128, generator=gen, device="cuda").to(BF16)
    a = rms_norm_fp8(x, None, EPS)
    got = torch.autograd.grad(prequantized_linear(a, weight), x, g)[0]
    assert a._runs is None  # no weight gradient, no token runs
    assert torch.equal(got, torch.autograd.grad(prequantized_linear(rms_norm(x, None, EPS), weight), x, g)[0])
    g = torch.randn(20, 256, generator=gen, device="cuda").to(BF16)
    through = torch.autograd.grad(rms_norm_fp8(x, None, EPS).dequantize(), x, g)[0]
    assert torch.equal(through, torch.autograd.grad(rms_norm(x, None, EPS), x, g)[0])


def test_modules_together():
    gen = torch.Generator(device="cuda").manual_seed(2)
    norm = FlexShardRMSNorm(256, eps=EPS, device="cuda", dtype=BF16)
    linear = FlexShardFloat8BlockwiseLinear(256, 128, bias=False, device="meta")
    del linear._parameters["weight"]
    linear.weight = _weight(128, 256, gen)
    x = torch.randn(9, 256, generator=gen, device="cuda").to(BF16)
    a, total = norm(x, x, fp8=True)
    assert torch.equal(linear(a), linear(norm(x, x)[0])) and torch.equal(total, x + x)


def test_changed_in_place_before_the_token_runs():
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(9, 256, generator=gen, device="cuda").to(BF16)
    a, total = rms_norm_fp8(x, None, EPS, residual=x)
    total.add_(1)
    with pytest.raises(RuntimeError, match="in place"):
        a.token_runs()


def test_no_rows():
    x = torch.zeros(0, 256, dtype=BF16, device="cuda", requires_grad=True)
    a, total = rms_norm_fp8(x, None, EPS, residual=x)
    assert a.shape == (0, 256) and a.q.shape == (0, 256) and a.dequantize().shape == (0, 256) and total.shape == (0, 256)


def test_another_gemm_object_is_refused():
    class Other:
        def forward(self, x, weight):
            return x

    gen = torch.Generator(device="cuda").manual_seed(4)
    a = rms_norm_fp8(torch.randn(4, 128, device="cuda"), None, EPS)
    with pytest.raises(TypeError, match="dequantize"):
        prequantized_linear(a, _weight(128, 128, gen), None, Other())
    with pytest.raises(ValueError, match="does not match"):
        prequantized_linear(a, _weight(128, 256, gen))


def test_captured_and_replayed():
    gen = torch.Generator(device="cuda").manual_seed(6)
    weight = _weight(256, 384, gen)
    x = torch.randn(60, 384, generator=gen, device="cuda").to(BF16).requires_grad_()
    w = torch.ones(384, device="cuda", requires_grad=True)
    g = torch.randn(60, 256, generator=gen, device="cuda").to(BF16)

    def once():
        a, total = rms_norm_fp8(x, w, EPS, residual=x)
        out = prequantized_linear(a, weight)
        return [out, total, *torch.autograd.grad([out, total], [x, w, weight], [g, total.detach()])]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for _ in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(60, 384, generator=gen, device="cuda").to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, once()))


def test_made_eagerly_and_read_by_two_graphs():
    """Neither graph may rely on token runs that the other one makes, nor eager work on either's."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    weight = _weight(256, 384, gen)
    x = torch.randn(60, 384, generator=gen, device="cuda").to(BF16)
    g = torch.randn(60, 256, generator=gen, device="cuda").to(BF16)
    a = rms_norm_fp8(x, torch.ones(384, device="cuda"), EPS)

    def once(activation):
        return torch.autograd.grad(prequantized_linear(activation, weight), weight, g)[0]

    want = once(rms_norm_fp8(x, torch.ones(384, device="cuda"), EPS))
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(once(a))
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[1], want) and torch.equal(once(a), want)
    for _ in range(3):
        outs[0].zero_()
        graphs[0].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want)


def test_weight_changed_before_the_token_runs():
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(9, 256, generator=gen, device="cuda").to(BF16)
    w = torch.ones(256, device="cuda")
    kept = rms_norm_fp8(x, w, EPS)
    with torch.no_grad():  # (no copy of the weight is kept)
        unkept = rms_norm_fp8(x, w, EPS)
    want = [t.clone() for t in rms_norm_fp8(x, w.clone(), EPS).token_runs()]
    w.mul_(2)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(kept.token_runs(), want))
    with pytest.raises(RuntimeError, match="in place"):
        unkept.token_runs()


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_in_the_backward(reentrant):
    """A checkpointed norm and its linear: the gradients of a run without one."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    weight = _weight(256, 384, gen)
    x = torch.randn(60, 384, generator=gen, device="cuda").to(BF16).requires_grad_()
    w = torch.ones(384, device="cuda", requires_grad=True)
    g = torch.randn(60, 256, generator=gen, device="cuda").to(BF16)

    def block(x):
        a, total = rms_norm_fp8(x, w, EPS, residual=x)
        return prequantized_linear(a, weight), total

    def grads(run):
        for leaf in (x, w, weight):
            leaf.grad = None
        out, total = run(x)
        torch.autograd.backward([out, total], [g, total.detach()])
        return [leaf.grad for leaf in (x, w, weight)]

    want = grads(block)
    got = grads(lambda x: torch.utils.checkpoint.checkpoint(block, x, use_reentrant=reentrant))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_made_in_a_checkpoint_and_read_behind_it():
    gen = torch.Generator(device="cuda").manual_seed(13)
    weight = _weight(256, 384, gen)
    x = torch.randn(60, 384, generator=gen, device="cuda").to(BF16).requires_grad_()
    w = torch.ones(384, device="cuda", requires_grad=True)
    g = torch.randn(60, 256, generator=gen, device="cuda").to(BF16)
    want = torch.autograd.grad(prequantized_linear(rms_norm_fp8(x, w, EPS), weight), (x, w, weight), g)
    a = torch.utils.checkpoint.checkpoint(rms_norm_fp8, x, w, EPS, use_reentrant=False)
    got = torch.autograd.grad(prequantized_linear(a, weight), (x, w, weight), g)
    assert all(torch.equal(s, t) for s, t in zip(got, want))


def test_read_on_another_stream():
    """Made on one stream, multiplied on another, dropped, and its memory asked for again meanwhile."""
    gen = torch.Generator(device="cuda").manual_seed(14)
    weight = _weight(256, 1024, gen)
    x = torch.randn(2000, 1024, generator=gen, device="cuda").to(BF16)
    w = torch.ones(1024, device="cuda")
    g = torch.randn(2000, 256, generator=gen, device="cuda").to(BF16)

    def once(a):
        out = prequantized_linear(a, weight)
        return [out.detach(), *torch.autograd.grad(out, weight, g)]

    want = once(rms_norm_fp8(x, w, EPS))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        busy = torch.randn(4096, 4096, device="cuda")
    for _ in range(3):
        a = rms_norm_fp8(x, w, EPS)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                busy = busy @ busy * 1e-3
            got = once(a)
        a.record_stream(side)
        del a
        for _ in range(4):
            rms_norm_fp8(x + 1, w * 2, EPS)
        side.synchronize()
        assert all(torch.equal(s, t) for s, t in zip(got, want))


@pytest.mark.parametrize("cols", [*range(1, 18), 121, 135, 255, 259, 383, 389, 513, 767, 771, 1285, 1530, 2305, 5113, 6001, 7161, 9001, 12290, 14001])
@pytest.mark.parametrize("dtype,stream", [(BF16, None), (BF16, F32), (F32, F32)])
def test_row_ends(dtype, stream, cols):
    """Every number of columns behind the last whole vector; the run that ends the row has its largest value last."""
    for rows in (3, 600):
        x, residual, w, _ = _make(rows, cols, dtype, stream)
        x[:, -1] = 40
        got, want = rms_norm_fp8(x, w, EPS, residual=residual), rms_norm(x, w, EPS, residual=residual)
        got, want = (got, want) if residual is None else (got[0], want[0])
        q, scales = hip_ops.act_quant_1x128(_quantized(want))
        assert _same(got.q, q) and torch.equal(got.scales, scales)
        assert not got.q.view(torch.uint8)[:, cols:].any()
