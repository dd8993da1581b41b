"""Calls of the 4-bit and expert entry points that have to be refused on the host, before a kernel sees their operands."""

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
