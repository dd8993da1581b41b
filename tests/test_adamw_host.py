"""What the optimizer's entry points refuse before anything reaches a GPU, and the
definition of its 8-bit states that the GPU tests compare with."""

import ctypes

import pytest
import torch
from adamw_definition import FIRST, SECOND, decode, dither, encode

from flex_shard_amd import _native, hip_ops
from flex_shard_amd.adamw import FlexShardAdamW, _check_state, grad_square_sum

OK, EINVAL, ENOTSUP = 0, -22, -95
SOMEWHERE = 1 << 20  # an aligned address that no refused call touches


def _message():
    return _native.lib().fsh_last_error().decode()


def _table(*values):
    return (ctypes.c_int64 * len(values))(*values)


def test_square_sum():
    lib = _native.lib()
    for tensor, status, word in (
        ((SOMEWHERE, -1, 0), EINVAL, "negative"), ((SOMEWHERE, 5, 3), EINVAL, "dtype"), ((SOMEWHERE, 5, -1), EINVAL, "dtype"),
        ((SOMEWHERE, 5, 1 << 40), EINVAL, "dtype"), ((0, 5, 0), EINVAL, "null"), ((SOMEWHERE + 1, 5, 0), ENOTSUP, "aligned"),
        ((SOMEWHERE + 2, 5, 1), ENOTSUP, "aligned"),
    ):
        assert lib.fsh_grad_square_sum(_table(SOMEWHERE, 8, 0, *tensor), 2, SOMEWHERE, SOMEWHERE, 1 << 20, None) == status
        assert word in _message() and _message().startswith("fsh_grad_square_sum")
    good = _table(SOMEWHERE, 8, 0)
    assert lib.fsh_grad_square_sum(good, -1, SOMEWHERE, SOMEWHERE, 64, None) == EINVAL
    assert lib.fsh_grad_square_sum(good, 1, None, SOMEWHERE, 64, None) == EINVAL
    assert lib.fsh_grad_square_sum(good, 1, SOMEWHERE + 4, SOMEWHERE, 64, None) == ENOTSUP
    many = _table(SOMEWHERE, 1 << 30, 0)
    assert lib.fsh_grad_square_sum(many, 1, SOMEWHERE, SOMEWHERE, 7, None) == EINVAL and "workspace" in _message()
    assert lib.fsh_grad_square_sum(many, 1, SOMEWHERE, None, 1 << 20, None) == EINVAL and "workspace" in _message()
    size = lib.fsh_grad_square_sum_workspace_bytes
    assert size(good, 1) == size(good, 0) == size(None, 1) == size(good, -1) == 0  # one workgroup does a few
    assert size(many, 1) == size(_table(SOMEWHERE, 1 << 40, 1), 1) == 8 * 4096


def _step(tensor=(), group=(), count=1, groups=1, square_sum=None, max_norm=0.0, workspace=SOMEWHERE, nbytes=1 << 20):
    values = [SOMEWHERE] * 7 + [1000, _native.DT_F32, _native.DT_F32, 8, 0]
    for at, value in dict(tensor).items():
        values[at] = value
    entry = dict(lr=1e-3, lr_dev=None, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1) | dict(group)
    table = (_native.AdamWGroup * 1)(tuple(entry.values()))
    return _native.lib().fsh_adamw_step(_table(*values), count, table, groups, square_sum, max_norm, workspace, nbytes, None)


@pytest.mark.parametrize(
    "arguments,status,word",
    [
        (dict(count=-1), EINVAL, "negative"), (dict(groups=0), ENOTSUP, "groups"), (dict(groups=17), ENOTSUP, "groups"),
        (dict(workspace=None), EINVAL, "null"), (dict(nbytes=8), EINVAL, "workspace"), (dict(workspace=SOMEWHERE + 8), EINVAL, "workspace"),
        (dict(square_sum=SOMEWHERE + 4), ENOTSUP, "sum"), (dict(max_norm=float("nan")), EINVAL, "max_norm"),
        (dict(group=dict(beta1=1.0)), EINVAL, "betas"), (dict(group=dict(beta2=-0.1)), EINVAL, "betas"),
        (dict(group=dict(beta2=float("nan"))), EINVAL, "betas"), (dict(group=dict(eps=-1.0)), EINVAL, "betas"),
        (dict(group=dict(lr_dev=SOMEWHERE + 2)), ENOTSUP, "learning rate"), (dict(tensor={7: -1}), EINVAL, "size"),
        (dict(tensor={11: 1}), EINVAL, "group"), (dict(tensor={11: -1}), EINVAL, "group"), (dict(tensor={8: 2}), EINVAL, "bf16"),
        (dict(tensor={9: 2}), EINVAL, "bf16"), (dict(tensor={10: 16}), EINVAL, "bits"), (dict(tensor={8: 1 << 33}), EINVAL, "bf16"),
        *((dict(tensor={at: 0}), EINVAL, "null") for at in range(7)),
        *((dict(tensor={at: SOMEWHERE + 2}), ENOTSUP, "aligned") for at in (0, 1, 4, 5, 6)),
        (dict(tensor={2: SOMEWHERE + 2, 10: 32}), ENOTSUP, "aligned"), (dict(tensor={7: 1 << 50}), ENOTSUP, "long"),
    ],
)
def test_step(arguments, status, word):
    assert _step(**arguments) == status
    assert word in _message() and _message().startswith("fsh_adamw_step")


def test_nothing_to_do():
    assert _step(count=0) == OK
    assert _native.lib().fsh_adamw_state_values(None, None, None, None, 0, None, None, 0, None) == OK
    assert _native.lib().fsh_adamw_step_workspace_bytes(-1) == 0
    assert ctypes.sizeof(_native.AdamWGroup) == 48


def test_state_values():
    call = _native.lib().fsh_adamw_state_values
    args = [SOMEWHERE] * 4 + [100, SOMEWHERE, SOMEWHERE, 0, None]
    for at, value, status in ((4, -1, EINVAL), (7, 3, EINVAL), (0, None, EINVAL), (6, None, EINVAL), (1, SOMEWHERE + 2, ENOTSUP), (5, SOMEWHERE + 1, ENOTSUP)):
        assert call(*args[:at], value, *args[at + 1 :]) == status, (at, value)


def test_there_is_no_cpu_path():
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="CPU"):
        FlexShardAdamW([p]).step()
    with pytest.raises(RuntimeError, match="CPU"):
        grad_square_sum([p.grad])
    p.grad = None
    assert FlexShardAdamW([p]).step() is None  # nothing to do


def test_a_refused_group_is_not_added():
    p, q = (torch.nn.Parameter(torch.zeros(4)) for _ in range(2))
    optimizer = FlexShardAdamW([p])
    with pytest.raises(ValueError):
        optimizer.add_param_group(dict(params=[q], betas=(0.9, 2.0)))
    assert len(optimizer.param_groups) == 1


# ---------------------------------------------------------------- the definition
@pytest.mark.parametrize("codes", [FIRST, SECOND])
def test_every_code_stands_for_itself(codes):
    """A block of all codes and its largest is encoded to the codes again, whatever the dither."""
    for sign in (0, 128) if codes == FIRST else (0,):
        code = torch.arange(codes + 1).add(torch.where(torch.arange(codes + 1) > 0, sign, 0)).to(torch.uint8)
        for part in code.split(127):
            part = torch.cat((part, torch.tensor([codes + sign], dtype=torch.uint8)))
            value = decode(part, torch.tensor([0.37]), codes)
            for t in (1, 2, 1000):
                again, scale = encode(value, t, codes)
                got = decode(again, scale, codes)
                # (0.37 times a code over 0.37 may miss it by a rounding, which the dither can take a step down)
                assert ((got - value).abs() <= value.abs() / 8).all() and scale[0] == torch.tensor(0.37)
            exact = decode(part, torch.ones(1), codes)
            assert torch.equal(encode(exact, 7, codes)[0], part)


@pytest.mark.parametrize("codes", [FIRST, SECOND])
def test_rounding_is_even_on_average(codes):
    """A value's mean over many steps and elements is the value: the dither's
    spread is a step of at most an eighth over 4000 draws, its error an eighth / sqrt(12 * 4000)."""
    for target in (0.7, 0.013, 3e-4):
        x = torch.full((128,), target)
        x[0] = 1.0
        values = torch.stack([decode(*encode(x, t, codes), codes)[1:] for t in range(1, 33)])
        assert abs(values.mean().item() / target - 1) < 5 * 0.125 / (12 * 32 * 127) ** 0.5
    if codes == FIRST:  # below the smallest code: that, or zero, as often as it takes
        x = torch.full((128,), 0.3 * 1.25 * 2.0**-16)
        x[0] = 1.0
        values = torch.stack([decode(*encode(x, t, codes), codes)[1:] for t in range(1, 33)])
        assert abs((values > 0).float().mean().item() - 0.3) < 5 * (0.21 / (32 * 127)) ** 0.5
    else:
        x = torch.full((128,), 1e-30)
        x[0] = 1.0
        assert (decode(*encode(x, 1, codes), codes) > 0).all()


def test_the_dither_is_uniform():
    for codes in (FIRST, SECOND):
        u = torch.cat([dither(1 << 16, t, codes) for t in (1, 2, 12345)]).double() / 2**32
        count = u.numel()
        assert abs(u.mean().item() - 0.5) < 5 / (12 * count) ** 0.5
        bins = torch.histc(u, 64, 0, 1)
        assert (bins - count / 64).abs().max() < 5 * (count / 64) ** 0.5


def test_tensors_that_overlap():
    """A parameter that is listed twice, one inside another, a shared step count: refused before anything is queued."""
    groups = (_native.AdamWGroup * 1)((1e-3, None, 0.9, 0.95, 1e-8, 0.1))

    def call(*tensors):  # (param, step, elements, dtype)
        rows = [(param, 1 << 40, 2 << 40, 3 << 40, 4 << 40, 5 << 40, step, n, dtype, _native.DT_F32, 32, 0) for param, step, n, dtype in tensors]
        return _native.lib().fsh_adamw_step(_table(*(v for row in rows for v in row)), len(rows), groups, 1, None, 0.0, 6 << 40, 1 << 20, None)

    far, steps = 1 << 30, 7 << 40
    for tensors in (
        ((SOMEWHERE, steps, 8, 1), (SOMEWHERE, steps + 4, 8, 1)),
        ((SOMEWHERE + 28, steps, 8, 1), (far, steps + 4, 8, 1), (SOMEWHERE, steps + 8, 8, 1)),
        ((SOMEWHERE, steps, 8, 0), (SOMEWHERE + 14, steps + 4, 1, 0)),
        ((SOMEWHERE, steps, 8, 1), (far, steps, 8, 1)),
        ((SOMEWHERE, steps, 0, 1), (far, steps, 0, 1)),
    ):
        assert call(*tensors) == EINVAL and "overlap" in _message(), tensors


def test_states_of_another_size_or_type():
    def state(**changed):
        return dict(
            step=torch.zeros((), dtype=torch.int32), exp_avg=torch.zeros(300, dtype=torch.uint8), exp_avg_sq=torch.zeros(300, dtype=torch.uint8),
            exp_avg_scale=torch.zeros(3), exp_avg_sq_scale=torch.zeros(3),
        ) | changed

    _check_state(state(), 300, 8, -1)  # (-1: on the CPU)
    _check_state(dict(step=torch.zeros((), dtype=torch.int32), exp_avg=torch.zeros(20, 15), exp_avg_sq=torch.zeros(20, 15)), 300, 32, -1)
    for name, value in (
        ("step", torch.zeros(())), ("exp_avg", torch.zeros(299, dtype=torch.uint8)), ("exp_avg", torch.zeros(300)),
        ("exp_avg_sq", torch.zeros(600, dtype=torch.uint8)[::2]), ("exp_avg_scale", torch.zeros(2)),
        ("exp_avg_sq_scale", torch.zeros(3, dtype=torch.float64)),
    ):
        with pytest.raises(ValueError, match=name):
            _check_state(state(**{name: value}), 300, 8, -1)
    with pytest.raises(ValueError, match="exp_avg"):
        _check_state(state(), 300, 32, -1)
    with pytest.raises(ValueError, match="step"):
        _check_state(state(), 300, 8, 0)


def test_states_of_torchs_own_are_loaded():
    p = torch.nn.Parameter(torch.ones(5))
    p.grad = torch.arange(5.0)
    for options in ({}, {"amsgrad": True}, {"maximize": True}):
        its = torch.optim.AdamW([p], lr=0.1, **options)
        its.step()
        mine = FlexShardAdamW([torch.nn.Parameter(torch.ones(5))], lr=0.5, state_bits=8)
        if options:
            with pytest.raises(NotImplementedError, match=next(iter(options))):
                mine.load_state_dict(its.state_dict())
            assert mine.param_groups[0]["state_bits"] == 8 and not mine.state
            continue
        mine.load_state_dict(its.state_dict())
        group = mine.param_groups[0]
        assert group["lr"] == 0.1 and group["state_bits"] == 32 and "state_bits" not in its.state_dict()["param_groups"][0]
        state = mine.state[group["params"][0]]
        assert torch.equal(state["exp_avg"], its.state[p]["exp_avg"]) and int(state["step"]) == 1 and state["step"].dtype == torch.int32
    bad = mine.state_dict()
    bad["param_groups"][0]["betas"] = (0.9, 1.0)
    with pytest.raises(ValueError, match="betas"):
        mine.load_state_dict(bad)


def _saved(bits):
    """A saved optimizer of two parameters, the first with states."""
    params = [torch.nn.Parameter(torch.ones(5)), torch.nn.Parameter(torch.ones(3))]
    optimizer = FlexShardAdamW(params, state_bits=bits)
    optimizer.state[params[0]] = optimizer._new_state(params[0], bits)
    optimizer.state[params[0]]["exp_avg"].copy_(torch.arange(5))
    optimizer.state[params[0]]["step"].fill_(7)
    return optimizer.state_dict()


@pytest.mark.parametrize("bits", [32, 8])
def test_load_hooks_see_the_states(bits):
    """A hook ahead of the loading gets all that was saved, and what it puts in its place is loaded; one behind
    it finds the states loaded."""
    params = [torch.nn.Parameter(torch.zeros(5)), torch.nn.Parameter(torch.zeros(3))]
    optimizer = FlexShardAdamW(params, state_bits=bits)
    seen = []

    def before(which, state_dict):
        seen.append((which, sorted(state_dict["state"]), sorted(state_dict["state"][0])))
        state = dict(state_dict["state"][0])
        state["exp_avg"] = state["exp_avg"] + 2  # (renamed, cut or converted, say)
        return {**state_dict, "state": {0: state}, "param_groups": [{**group, "lr": 0.25} for group in state_dict["param_groups"]]}

    def behind(which):
        seen.append((which, int(which.state[params[0]]["step"]), which.state[params[0]]["exp_avg"].tolist()))

    optimizer.register_load_state_dict_pre_hook(before)
    optimizer.register_load_state_dict_post_hook(behind)
    saved = _saved(bits)
    names = sorted(saved["state"][0])
    for _ in range(2):
        optimizer.load_state_dict(saved)
        assert seen == [(optimizer, [0], names), (optimizer, 7, [2, 3, 4, 5, 6])]
        state = optimizer.state[params[0]]
        assert state["exp_avg"].dtype == (torch.uint8 if bits == 8 else torch.float32) and state["step"].dtype == torch.int32
        assert optimizer.param_groups[0]["lr"] == 0.25 and not optimizer.state.get(params[1])
        seen.clear()
    assert saved["state"][0]["exp_avg"].tolist() == [0, 1, 2, 3, 4]


def test_what_else_was_saved_is_loaded():
    """States of other names, of no parameter, and of a parameter that has none yet."""
    params = [torch.nn.Parameter(torch.zeros(5)), torch.nn.Parameter(torch.zeros(3))]
    optimizer = FlexShardAdamW(params)
    saved = _saved(32)
    saved["state"][0]["note"] = torch.tensor([4.0])
    saved["state"][1] = {}
    saved["state"]["all"] = torch.tensor(3.0)
    optimizer.load_state_dict(saved)
    assert optimizer.state["all"].item() == 3 and not optimizer.state.get(params[1])
    state = optimizer.state[params[0]]
    assert state["note"].item() == 4 and int(state["step"]) == 7 and state["exp_avg"].tolist() == [0, 1, 2, 3, 4]
    assert state["exp_avg"] is not saved["state"][0]["exp_avg"] and state["step"].dtype == torch.int32


def test_a_refused_loading_changes_nothing():
    params = [torch.nn.Parameter(torch.zeros(5)), torch.nn.Parameter(torch.zeros(3))]
    optimizer = FlexShardAdamW(params, lr=0.5)
    optimizer.load_state_dict(_saved(32) | {"param_groups": [{**_saved(32)["param_groups"][0], "lr": 0.5}]})
    kept = optimizer.state[params[0]]
    calls = []
    optimizer.register_load_state_dict_post_hook(calls.append)
    other = _saved(32)
    other["state"][0]["exp_avg_sq"] = torch.zeros(4)
    fewer = _saved(32)
    fewer["param_groups"][0]["params"] = [0]
    for bad in (other, fewer):
        with pytest.raises(ValueError):
            optimizer.load_state_dict(bad)
        assert optimizer.state[params[0]] is kept and optimizer.param_groups[0]["lr"] == 0.5 and not calls


def _many_groups(count, params, group=()):
    """The tables of as many tensors of 8 fp32 elements, a group each; ``params``: addresses other than their own."""
    rows = [[(1 << 20) * (i + 1) + (at << 30) for at in range(7)] + [8, _native.DT_F32, _native.DT_F32, 8, i] for i in range(count)]
    for at, address in params.items():
        rows[at][0] = address
    groups = [(1e-3, None, 0.9, 0.95, 1e-8, 0.1)] * count
    for at, values in dict(group).items():
        groups[at] = values
    return rows, groups


@pytest.mark.parametrize(
    "params,group,word",
    [
        ({18: (1 << 20) + 28}, {}, "overlap"), ({18: (1 << 20) * 2 - 28}, {}, "overlap"), ({19: 0}, {}, "null"), ({19: (1 << 30) - 2}, {}, "aligned"),
        ({}, {19: (1e-3, None, 1.0, 0.95, 1e-8, 0.1)}, "group 19"), ({}, {19: (1e-3, SOMEWHERE + 2, 0.9, 0.95, 1e-8, 0.1)}, "group 19"),
    ],
)
def test_groups_of_several_calls_are_checked_together(params, group, word, monkeypatch):
    """Twenty groups: what is wrong with the last is found before the first call, and so is what overlaps between calls."""
    rows, groups = _many_groups(20, params, group)
    table = _table(*(v for row in rows for v in row))
    check = _native.lib().fsh_adamw_check
    of_groups = (_native.AdamWGroup * 20)(*groups)
    assert check(table, 20, of_groups, 20) in (EINVAL, ENOTSUP)
    assert word in _message() and _message().startswith("fsh_adamw_check")
    queued = []
    monkeypatch.setattr(hip_ops, "_queue", lambda *args: queued.append(args))
    cpu = torch.device("cpu")
    with pytest.raises(RuntimeError, match=word):
        hip_ops.adamw_step([v for row in rows for v in row], groups, cpu)
    assert not queued


def test_groups_of_several_calls(monkeypatch):
    rows, groups = _many_groups(40, {})
    groups = [(1e-3 * (i + 1), *group[1:]) for i, group in enumerate(groups)]
    rows = rows[::2] + [rows[i] for i in range(1, 40, 2) if i not in (17, 19)]  # (in any order, two without tensors)
    queued = []
    monkeypatch.setattr(hip_ops, "_queue", lambda *args: queued.append(args))
    hip_ops.adamw_step([v for row in rows for v in row], groups, torch.device("cpu"))
    got = {}
    for entry, _, table, count, of_groups, group_count, *_ in queued:
        assert entry == "fsh_adamw_step" and group_count <= _native.ADAMW_GROUPS and len(table) == 12 * count
        for at in range(0, 12 * count, 12):
            got[tuple(table[at : at + 11])] = of_groups[table[at + 11]].lr
    assert len(queued) == 3 and got == {tuple(row[:11]): groups[row[11]][0] for row in rows}
    check = _native.lib().fsh_adamw_check
    assert check(None, 0, None, 0) == OK and check(None, 1, None, 0) == EINVAL and check(None, -1, None, 0) == EINVAL


# 0 parameter, 1 gradient, 2 and 3 moments, 4 and 5 scales, 6 step count
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize(
    "at,over,status",
    [
        *(((1, one), (0, other), EINVAL) for one in (0, 2, 3, 6) for other in (0, 2, 3, 6)),
        *(((1, 1), (0, other), EINVAL) for other in (0, 2, 3, 6)), *(((0, one), (0, other), EINVAL) for one in (2, 3, 6) for other in (0, 1)),
        ((0, 3), (0, 2), EINVAL), ((1, 1), (0, 1), OK), ((0, 1), (0, 0), OK),
    ],
)
def test_states_and_gradients_that_overlap(bits, at, over, status):
    """A step's parameters, states and step counts lie apart, and no gradient lies over them; one gradient may serve two."""
    rows, groups = _many_groups(2, {})
    for row in rows:
        row[10] = bits
    rows[at[0]][at[1]] = rows[over[0]][over[1]]
    _expect(rows, groups, status)


@pytest.mark.parametrize("one", range(7))
def test_scales_that_overlap(one):
    for scale in (4, 5):
        rows, groups = _many_groups(2, {})
        for row in rows:
            row[7] = 300  # three blocks
        rows[1][scale] = rows[0][one] - 8 if one not in (2, 3) else rows[0][one] + 296
        _expect(rows, groups, EINVAL)
        rows[1][scale] = rows[0][one] - 12
        _expect(rows, groups, OK)
    rows[1][10] = rows[0][10] = 32  # states that have none
    rows[1][4] = rows[1][5] = rows[0][4]
    _expect(rows, groups, OK)


def _expect(rows, groups, status):
    of_groups = (_native.AdamWGroup * len(groups))(*groups)
    assert _native.lib().fsh_adamw_check(_table(*(v for row in rows for v in row)), len(rows), of_groups, len(groups)) == status, rows
    assert status == OK or "overlap" in _message()


def test_a_workspace_over_a_state():
    rows, groups = _many_groups(1, {})
    of_groups = (_native.AdamWGroup * 1)(*groups)
    for at in range(7):
        table = _table(*rows[0])
        assert _native.lib().fsh_adamw_step(table, 1, of_groups, 1, None, 0.0, rows[0][at] - 32, 1 << 20, None) == EINVAL and "overlap" in _message()


def test_state_values_over_their_codes():
    call, far = _native.lib().fsh_adamw_state_values, [SOMEWHERE + (i << 20) for i in range(6)]
    for first, second in ((far[0], far[5]), (far[4], far[2] - 198), (far[1] - 196, far[5]), (far[4], far[4] + 198)):
        assert call(*far[:4], 100, first, second, _native.DT_BF16, None) == EINVAL and "overlaps" in _message()
