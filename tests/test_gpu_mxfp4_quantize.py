"""The 4-bit quantizers and the way back against the definition, bit for bit."""

import pytest
import torch
from mxfp4_definition import quantize, unpack, values

from flex_shard_amd import hip_ops
from flex_shard_amd.mxfp4 import mxfp4_quantize, mxfp4_quantize_both, mxfp4_quantize_transposed, quantize_mxfp4_weight

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _random(rows, cols, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=gen) * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=gen).float())
    return x.to(dtype)


def _assert_matrix(matrix, x):
    """``matrix`` is the definition's quantization of the CPU matrix ``x``."""
    codes, byte = quantize(x)
    got_codes, got_byte = unpack(*matrix.pair)
    assert torch.equal(got_byte, byte)
    finite = (byte != 255).repeat_interleave(32, dim=1)
    assert torch.equal(torch.where(finite, got_codes, 0), torch.where(finite, codes, 0))
    want = values(codes, byte, x.shape[1])
    for dtype in DTYPES:
        got = matrix.dequantize(dtype)
        assert got.dtype == dtype and torch.equal(got.cpu().nan_to_num(7.5), want.to(dtype).nan_to_num(7.5))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_16_bit_value(device, dtype):
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
    finite = bits[torch.isfinite(bits)]
    ordered = finite[finite.float().abs().argsort()]
    # runs of neighbours; runs whose first element is up to 2**8 times the others
    spread = ordered.view(-1, 16).repeat_interleave(2, dim=0).flatten().view(-1, 32).clone()
    spread[:, 0] = (spread[:, 0].float() * 2.0 ** (torch.arange(len(spread)) % 9)).to(dtype)
    spread = torch.where(torch.isfinite(spread), spread, 0.0)
    for x in (ordered.view(-1, 256), spread.view(-1, 32)):
        _assert_matrix(mxfp4_quantize(x.to(device)), x)
        _assert_matrix(mxfp4_quantize_transposed(x.t().contiguous().to(device)), x)


def test_fp32_values_at_and_beside_every_tie(device):
    middles = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 6.0, 2.0, 4.0])
    near = torch.cat([middles, torch.nextafter(middles, torch.tensor(0.0)), torch.nextafter(middles, torch.tensor(99.0))])
    run = torch.cat([near[:31], torch.tensor([4.0])])
    exponents = torch.arange(-126, 125, 5).float()
    x = run * torch.exp2(exponents)[:, None]
    x = torch.cat([x, -x])
    assert torch.isfinite(x).all()
    _assert_matrix(mxfp4_quantize(x.to(device)), x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (31, 33), (130, 256), (128, 257), (257, 130), (5, 1000), (300, 520)])
def test_sizes(device, rows, cols, dtype):
    x = _random(rows, cols, dtype, rows * 1000 + cols)
    on_gpu = x.to(device)
    _assert_matrix(mxfp4_quantize(on_gpu), x)
    _assert_matrix(mxfp4_quantize_transposed(on_gpu), x.t())
    along, across = mxfp4_quantize_both(on_gpu)
    _assert_matrix(along, x)
    _assert_matrix(across, x.t())


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_unaligned_rows(device, dtype):
    whole = _random(70, 301, dtype, 3)
    on_gpu = whole.to(device)
    for part in (slice(1, 290), slice(8, 264), slice(3, 4)):
        x = on_gpu[:, part]
        _assert_matrix(mxfp4_quantize(x), whole[:, part])
        along, across = mxfp4_quantize_both(x)
        _assert_matrix(along, whole[:, part])
        _assert_matrix(across, whole[:, part].t())
    _assert_matrix(mxfp4_quantize(on_gpu.t()), whole.t())  # columns of another matrix
    _assert_matrix(mxfp4_quantize(on_gpu[:1].expand(40, 301)), whole[:1].expand(40, 301))


@pytest.mark.parametrize("dtype", DTYPES)
def test_zeros_infinities_and_nans_stay_in_their_runs(device, dtype):
    x = _random(64, 320, dtype, 4)
    x[2] = 0.0
    x[3, 32:64] = -0.0
    x[5, 40] = float("inf")
    x[6, 100] = float("nan")
    x[7, 319] = -float("inf")
    x[9] = torch.finfo(dtype).max
    x[10] = torch.finfo(dtype).smallest_normal / 64  # subnormal (or zero) throughout
    _assert_matrix(mxfp4_quantize(x.to(device)), x)
    along, across = mxfp4_quantize_both(x.to(device))
    _assert_matrix(along, x)
    _assert_matrix(across, x.t())


@pytest.mark.parametrize("dtype", DTYPES)
def test_stacked_weights(device, dtype):
    w = _random(3 * 65, 290, dtype, 5).view(3, 65, 290)
    weight = quantize_mxfp4_weight(w.to(device), transposed=True)
    _assert_matrix(weight.matrix, w.reshape(-1, 290))
    _assert_matrix(weight.transposed, w.transpose(1, 2).reshape(-1, 65))
    assert weight.shape == (3, 65, 290) and weight.dtype == dtype


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 40), (128, 64), (1000, 129)])
def test_column_sums(device, rows, cols, dtype):
    x = _random(rows, cols, dtype, 6)
    _, _, sums = hip_ops.mxfp4_quantize(x.to(device), rows=False, columns=True, column_sums=True)
    assert sums.shape == (-(-rows // 128), cols)
    got = hip_ops.sum_runs(sums, torch.float32).cpu().double()
    want, size = x.double().sum(dim=0), x.double().abs().sum(dim=0)
    assert ((got - want).abs() <= rows * 2.0**-24 * size).all()


@pytest.mark.parametrize("gathered", [False, True])
def test_segments_are_padded_with_zeros(device, gathered):
    lengths = [0, 3, 256, 0, 300, 1, 0]
    top_k, tokens = 2, 300
    rows = tokens * top_k
    used = sum(lengths)
    x = _random(tokens if gathered else rows, 75, torch.bfloat16, 7)
    gen = torch.Generator().manual_seed(1)
    source = torch.randperm(rows, generator=gen).to(torch.int32)
    source[used:] = -1
    offsets = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
    padded = torch.tensor([0] + [-(-n // 256) * 256 for n in lengths]).cumsum(0).to(torch.int32)
    row_form, column_form = hip_ops.mxfp4_quantize_segments(
        x.to(device), offsets.to(device), padded.to(device), 1280, choices=rows, source=source.to(device) if gathered else None,
        top_k=top_k, rows=not gathered,
    )
    sorted_rows = x[source[:used].long() // top_k] if gathered else x[:used]
    got_codes, got_byte = unpack(*column_form)
    for e, n in enumerate(lengths):
        codes, byte = quantize(sorted_rows[offsets[e] : offsets[e] + n].t())
        begin, end = int(padded[e]), int(padded[e + 1])
        assert torch.equal(got_codes[:, begin:end], codes) and torch.equal(got_byte[:, begin // 32 : end // 32], byte)
    if not gathered:
        got_codes, got_byte = unpack(row_form[0][:used], row_form[1][:, :used].contiguous())
        codes, byte = quantize(sorted_rows)
        assert torch.equal(got_codes, codes) and torch.equal(got_byte, byte)


def test_empty_matrices(device):
    for shape in ((0, 64), (5, 0)):
        matrix = mxfp4_quantize(torch.empty(shape, device=device))
        assert matrix.rows == shape[0] and matrix.dequantize().shape == shape


def test_refusals(device):
    x = torch.randn(8, 64, device=device)
    with pytest.raises(RuntimeError, match="no CPU path"):
        mxfp4_quantize(x.cpu())
    with pytest.raises(NotImplementedError):
        mxfp4_quantize(x.double())
    with pytest.raises(ValueError, match="matrix"):
        mxfp4_quantize(x[0])
    with pytest.raises(ValueError, match="rows"):
        hip_ops.mxfp4_quantize(x.t())
    with pytest.raises(ValueError):
        hip_ops.mxfp4_quantize(x, rows=False)
    with pytest.raises(ValueError, match="contiguous"):
        hip_ops.mxfp4_quantize(torch.randn(2, 8, 64, device=device).transpose(1, 2))
    matrix = mxfp4_quantize(x)
    with pytest.raises(ValueError, match="columns"):
        hip_ops.mxfp4_dequantize(*matrix.pair, 300, torch.float32)
    with pytest.raises(ValueError, match="out must be"):
        hip_ops.mxfp4_dequantize(*matrix.pair, 64, torch.float32, out=torch.empty(8, 64, device=device, dtype=torch.bfloat16))
