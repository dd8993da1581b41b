"""Calls of the 4-bit and expert entry points that have to be refused on the host, before a kernel sees their operands."""

import ctypes

import pytest

from flex_shard_amd import _native

OK, EINVAL, ENOTSUP = 0, -22, -95
SOMEWHERE = 1 << 20  # an aligned address that no refused call touches


def _message():
    return _native.lib().fsh_last_error().decode()


def test_combine_of_fp32_rows():
    call = _native.lib().fsh_expert_combine_f32
    args = [SOMEWHERE, SOMEWHERE, SOMEWHERE, 1, 4, 2, 8, 0, SOMEWHERE, None]
    for at, value, status in ((4, -1, EINVAL), (5, 0, EINVAL), (5, 65, ENOTSUP), (6, -1, EINVAL), (7, 5, EINVAL), (3, 9, EINVAL),
                              (0, None, EINVAL), (1, None, EINVAL), (8, None, EINVAL), (0, SOMEWHERE + 2, ENOTSUP), (8, SOMEWHERE + 1, ENOTSUP)):
        assert call(*args[:at], value, *args[at + 1 :]) == status, (at, value)
        assert _message().startswith("fsh_expert_combine_f32")
    assert call(SOMEWHERE, SOMEWHERE, None, 1, 0, 2, 8, 0, SOMEWHERE, None) == OK


def _product(**fields):
    q = _native.MxFp4Product()
    for name in ("a_dev", "a_scales_dev", "b_dev", "b_scales_dev", "out_dev"):
        setattr(q, name, SOMEWHERE)
    q.m, q.n, q.k, q.a_rows, q.b_rows, q.ldo, q.top_k = 8, 16, 256, 8, 16, 16, 1
    for name, value in fields.items():
        setattr(q, name, value)
    return ctypes.byref(q)


BIAS_F32 = _native.MXFP4_BIAS_F32


@pytest.mark.parametrize(
    "fields,status,word",
    [
        (dict(mode=BIAS_F32 + 1, experts=1, offsets_dev=SOMEWHERE), EINVAL, "mode"),
        (dict(mode=BIAS_F32 + 2, experts=1, offsets_dev=SOMEWHERE), EINVAL, "mode"),
        (dict(mode=2 * BIAS_F32), EINVAL, "mode"),
        (dict(mode=BIAS_F32, bias_dev=SOMEWHERE + 2), ENOTSUP, "aligned"),
    ],
)
def test_fp32_bias(fields, status, word):
    assert _native.lib().fsh_mxfp4_gemm(_product(**fields), None) == status
    assert word in _message()


def test_fp32_bias_of_a_few_rows():
    call = _native.lib().fsh_mxfp4_linear
    product = _product(m=2, a_rows=2, mode=BIAS_F32, bias_dev=SOMEWHERE + 2)
    assert call(SOMEWHERE, 0, 2, 256, product, 256, None, 0, None) == ENOTSUP and "aligned" in _message()


@pytest.mark.parametrize("experts", [1025, 1 << 20])
def test_more_experts_than_a_tile_has_a_table_for(experts):
    fields = dict(mode=_native.MXFP4_ROWS, experts=experts, offsets_dev=SOMEWHERE, b_rows=16 * experts)
    assert _native.lib().fsh_mxfp4_gemm(_product(**fields), None) == ENOTSUP and "1024 experts" in _message()
    # (ahead of the quantizer's launch)
    status = _native.lib().fsh_mxfp4_linear(SOMEWHERE, 0, 8, 256, _product(**fields), 256, SOMEWHERE, 1 << 20, None)
    assert status == ENOTSUP and "1024 experts" in _message()
    assert _native.lib().fsh_mxfp4_gemm_tiles(8, 16, 256, _native.MXFP4_ROWS, experts) == ENOTSUP
    assert _native.lib().fsh_mxfp4_gemm_tiles(8, 16, 256, _native.MXFP4_ROWS, _native.MAX_EXPERTS) >= 0


@pytest.mark.parametrize(
    "fields,in_dim,status,word",
    [(dict(m=-1), 256, EINVAL, "negative"), (dict(m=2, n=-100, ldo=16), 256, EINVAL, "negative"), (dict(m=2, k=0), 0, ENOTSUP, "positive"),
     (dict(m=8, k=0), 0, ENOTSUP, "positive"), (dict(m=2, k=-256), 256, EINVAL, "in_dim")],
)
def test_linear_sizes(fields, in_dim, status, word):
    call = _native.lib().fsh_mxfp4_linear
    assert call(SOMEWHERE, 0, 8, 256, _product(**fields), in_dim, SOMEWHERE, 1 << 20, None) == status
    assert word in _message()


@pytest.mark.parametrize("m", [2, 8])
def test_linear_of_no_rows_has_no_outputs(m):
    call = _native.lib().fsh_mxfp4_linear
    assert call(SOMEWHERE, 0, 0, 256, _product(m=m), 256, SOMEWHERE, 1 << 20, None) == EINVAL  # outputs that nothing would write
    assert call(SOMEWHERE, 0, 0, 256, _product(m=0), 256, None, 0, None) == OK
