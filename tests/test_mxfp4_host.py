"""What the 4-bit and expert entry points refuse before anything reaches a GPU,
and the definition that the GPU tests compare with."""

import ctypes

import pytest
import torch
from mxfp4_definition import quantize, through, unpack

from flex_shard_amd import _native
from flex_shard_amd.experts import ExpertRouting, route_tokens
from flex_shard_amd.mxfp4 import mxfp4_linear, mxfp4_quantize

OK, EINVAL, ENOTSUP = 0, -22, -95
SOMEWHERE = 1 << 20  # an aligned address that no refused call touches


def _message():
    return _native.lib().fsh_last_error().decode()


def test_struct_size():
    assert ctypes.sizeof(_native.MxFp4Product) == 8 * 8 + 6 * 8 + 4 * 4


def test_quantizer_arguments():
    lib = _native.lib()
    call = lib.fsh_mxfp4_quantize
    assert call(None, 0, 1, 0, 5, 5, None, None, None, None, None, None) == OK  # nothing to do
    assert call(SOMEWHERE, 0, 1, -1, 5, 5, None, None, None, None, None, None) == EINVAL
    assert call(SOMEWHERE, 7, 1, 4, 5, 5, SOMEWHERE, SOMEWHERE, None, None, None, None) == EINVAL and "dtype" in _message()
    assert call(SOMEWHERE, 0, 1, 4, 5, 5, None, None, None, None, None, None) == EINVAL and "no output" in _message()
    assert call(SOMEWHERE, 0, 1, 4, 5, 5, SOMEWHERE, None, None, None, None, None) == EINVAL and "go together" in _message()
    assert call(None, 0, 1, 4, 5, 5, SOMEWHERE, SOMEWHERE, None, None, None, None) == EINVAL and "null" in _message()
    assert call(SOMEWHERE, 0, 1, 4, 5, 4, SOMEWHERE, SOMEWHERE, None, None, None, None) == EINVAL and "ldx" in _message()
    assert call(SOMEWHERE, 0, 1, 4, 5, 5, SOMEWHERE + 8, SOMEWHERE, None, None, None, None) == ENOTSUP
    assert call(SOMEWHERE, 0, 2, 4, 5, 6, None, None, SOMEWHERE, SOMEWHERE, None, None) == ENOTSUP and "stack" in _message()
    assert call(SOMEWHERE, 0, 1, 4, 5, 5, SOMEWHERE, SOMEWHERE, None, None, SOMEWHERE, None) == EINVAL and "sums" in _message()
    segments = lib.fsh_mxfp4_quantize_segments
    args = [SOMEWHERE, 0, 300, 5, 5, SOMEWHERE, SOMEWHERE, 2, None, 1, None, None, SOMEWHERE, SOMEWHERE, 512, None]
    for at, value, word in ((7, 0, "expert"), (14, 256, "padded_rows"), (14, 500, "padded_rows"), (5, None, "null")):
        assert segments(*args[:at], value, *args[at + 1 :]) == EINVAL and word in _message()
    gathered = args.copy()
    gathered[8] = gathered[10] = gathered[11] = SOMEWHERE
    assert segments(*gathered) == EINVAL and "row form" in _message()
    assert lib.fsh_mxfp4_dequantize(SOMEWHERE, SOMEWHERE, 4, 5, SOMEWHERE, 0, 4, None) == EINVAL
    assert lib.fsh_mxfp4_dequantize(SOMEWHERE, SOMEWHERE, 4, 5, SOMEWHERE, 9, 5, None) == EINVAL
    assert lib.fsh_sum_runs(None, 3, 5, SOMEWHERE, 0, None) == EINVAL


def _product(**fields):
    q = _native.MxFp4Product()
    for name in ("a_dev", "a_scales_dev", "b_dev", "b_scales_dev", "out_dev"):
        setattr(q, name, SOMEWHERE)
    q.m, q.n, q.k, q.a_rows, q.b_rows, q.ldo, q.top_k = 8, 16, 256, 8, 16, 16, 1
    for name, value in fields.items():
        setattr(q, name, value)
    return ctypes.byref(q)


@pytest.mark.parametrize(
    "fields,status,word",
    [
        (dict(m=-1), EINVAL, "negative"),
        (dict(mode=5), EINVAL, "mode"),
        (dict(mode=1), EINVAL, "expert"),
        (dict(mode=1, experts=2), EINVAL, "offsets"),
        (dict(mode=1, experts=2, offsets_dev=SOMEWHERE), EINVAL, "too few"),
        (dict(mode=1, experts=1, offsets_dev=SOMEWHERE, top_k=0), EINVAL, "top_k"),
        (dict(mode=1, experts=1, offsets_dev=SOMEWHERE, bias_dev=SOMEWHERE), ENOTSUP, "bias"),
        (dict(mode=2, experts=1, offsets_dev=SOMEWHERE, ldo=20), EINVAL, "contiguous"),
        (dict(source_dev=SOMEWHERE), EINVAL, "gathered"),
        (dict(out_dtype=9), EINVAL, "dtype"),
        (dict(a_dev=None), EINVAL, "null"),
        (dict(k=128), ENOTSUP, "multiple of 256"),
        (dict(k=0), ENOTSUP, "multiple of 256"),
        (dict(k=1 << 31), ENOTSUP, "2^31"),
        (dict(a_rows=7), EINVAL, "too few"),
        (dict(b_rows=15), EINVAL, "too few"),
        (dict(ldo=15), EINVAL, "ldo"),
        (dict(a_dev=SOMEWHERE + 8), ENOTSUP, "aligned"),
        (dict(out_dtype=1, out_dev=SOMEWHERE + 2), ENOTSUP, "aligned"),
        (dict(k=1 << 26), ENOTSUP, "4 GiB"),
        (dict(mode=1, experts=1, offsets_dev=SOMEWHERE, source_dev=SOMEWHERE, a_rows=1 << 27), ENOTSUP, "4 GiB"),
    ],
)
def test_product_arguments(fields, status, word):
    assert _native.lib().fsh_mxfp4_gemm(_product(**fields), None) == status
    assert word in _message()


def test_product_of_nothing():
    assert _native.lib().fsh_mxfp4_gemm(None, None) == EINVAL
    assert _native.lib().fsh_mxfp4_gemm(_product(m=0), None) == OK
    assert _native.lib().fsh_mxfp4_gemm(_product(n=0), None) == OK


def test_expert_arguments():
    lib = _native.lib()
    route = lib.fsh_expert_route
    assert route(SOMEWHERE, 3, 8, 2, *[SOMEWHERE] * 4, None, 0, None) == EINVAL and "bytes" in _message()
    assert route(SOMEWHERE, 8, 8, 0, *[SOMEWHERE] * 4, None, 0, None) == EINVAL
    assert route(SOMEWHERE, 8, 8, 1025, *[SOMEWHERE] * 4, None, 0, None) == ENOTSUP
    assert route(SOMEWHERE + 4, 8, 8, 2, *[SOMEWHERE] * 4, None, 0, None) == ENOTSUP
    assert route(None, 8, 8, 2, *[SOMEWHERE] * 4, None, 0, None) == EINVAL
    assert route(SOMEWHERE, 8, (1 << 31) - 300, 2, *[SOMEWHERE] * 4, None, 0, None) == ENOTSUP
    assert lib.fsh_expert_route_workspace_bytes(100, 8) == 0
    need = lib.fsh_expert_route_workspace_bytes(100000, 8)
    assert need > 0 and route(SOMEWHERE, 8, 100000, 8, *[SOMEWHERE] * 4, SOMEWHERE, need - 1, None) == EINVAL
    for call, args in (
        (lib.fsh_expert_dispatch, [SOMEWHERE, SOMEWHERE, SOMEWHERE, 2, 4, 2, 8, 0, SOMEWHERE, None]),
        (lib.fsh_expert_combine, [SOMEWHERE, SOMEWHERE, SOMEWHERE, 1, 4, 2, 8, 0, SOMEWHERE, None]),
        (lib.fsh_expert_combine_backward, [SOMEWHERE, SOMEWHERE, SOMEWHERE, SOMEWHERE, 2, SOMEWHERE, 1, 4, 2, 8, 0, SOMEWHERE, SOMEWHERE, None]),
    ):
        first = len(args) - (6 if call is not lib.fsh_expert_combine_backward else 7)  # of tokens, top_k, width, dtype
        for at, value, status in ((0, -1, EINVAL), (1, 0, EINVAL), (1, 65, ENOTSUP), (2, -1, EINVAL), (3, 5, EINVAL)):
            changed = args.copy()
            changed[first + at] = value
            assert call(*changed, ) == status, (call, at, value)
        assert call(None, *args[1:]) == EINVAL


def test_nothing_runs_off_the_gpu():
    with pytest.raises(RuntimeError, match="no CPU path"):
        mxfp4_quantize(torch.zeros(2, 32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        mxfp4_linear(torch.zeros(2, 32), torch.zeros(4, 32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        route_tokens(torch.zeros(2, 1, dtype=torch.int64), 4)


def test_padded_rows_hold_every_routing():
    for experts in (1, 2, 7):
        for rows in (1, 2, 255, 256, 257, 600):
            routing = ExpertRouting(experts, torch.zeros(rows, 1), torch.zeros(1), torch.zeros(rows), torch.zeros(1))
            worst = 0
            for first in {0, 1, min(rows, 256), min(rows, 257), rows}:
                lengths = [first] + [0] * (experts - 1)
                for i in range(rows - first):
                    lengths[(1 + i) % experts] += 1
                worst = max(worst, sum(-(-n // 256) * 256 for n in lengths))
            assert worst <= routing.padded_rows and routing.padded_rows % 256 == 0 and routing.padded_rows >= rows


def test_definition():
    x = torch.tensor([[1.0, -0.25, 0.75, 0.125, 0.375, 1.75, 1.25, 0.0625] + [0.0] * 25])
    codes, byte = quantize(x)
    assert byte[0, :3].tolist() == [125, 0, 0]
    # 4 x 0.25 ... : scaled by 4 these are 4, -1, 3, 0.5, 1.5, 7, 5, 0.25
    assert codes[0, :8].tolist() == [6, 10, 5, 1, 3, 7, 6, 0]
    assert through(x)[0, :8].tolist() == [1.0, -0.25, 0.75, 0.125, 0.375, 1.5, 1.0, 0.0]
    data = (codes[:, ::2] + 16 * codes[:, 1::2]).to(torch.uint8)
    scales = byte.to(torch.uint8).view(1, -1, 8).permute(1, 0, 2)
    again = unpack(data, scales)
    assert torch.equal(again[0], codes) and torch.equal(again[1], byte)
