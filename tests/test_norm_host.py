"""What the norms' entry points refuse before anything reaches a GPU."""

import ctypes

import pytest
import torch

from flex_shard_amd import _native
from flex_shard_amd.norms import FlexShardRMSNorm, convert_to_flex_shard_rms_norm, rms_norm, rms_norm_fp8

OK, EINVAL, ENOTSUP = 0, -22, -95
SOMEWHERE = 1 << 20  # an aligned address that no refused call touches
BF16, F32, F16 = _native.DT_BF16, _native.DT_F32, _native.DT_F16


def _message():
    return _native.lib().fsh_last_error().decode()


def test_struct_sizes():
    assert ctypes.sizeof(_native.Norm) == 7 * 8 + 4 * 8 + 6 * 4
    assert ctypes.sizeof(_native.NormGradient) == 9 * 8 + 6 * 8 + 4 * 4


def _norm(**fields):
    q = _native.Norm()
    for name in ("x_dev", "residual_dev", "weight_dev", "total_dev", "out_dev", "scales_dev", "rstd_dev"):
        setattr(q, name, SOMEWHERE)
    q.rows, q.cols, q.ldx, q.ldr, q.eps = 4, 100, 100, 100, 1e-6
    for name, value in fields.items():
        setattr(q, name, value)
    return ctypes.byref(q)


@pytest.mark.parametrize(
    "fields,status,word",
    [
        (dict(rows=-1), EINVAL, "negative"), (dict(cols=-1), EINVAL, "negative"), (dict(x_dtype=3), EINVAL, "dtype"),
        (dict(x_dtype=-1), EINVAL, "dtype"), (dict(weight_dtype=9), EINVAL, "dtype"), (dict(form=2), EINVAL, "form"),
        (dict(residual_dtype=F16), EINVAL, "residual"), (dict(x_dtype=F32), EINVAL, "residual"),
        (dict(eps=-1.0), EINVAL, "eps"), (dict(eps=float("nan")), EINVAL, "eps"), (dict(x_dev=None), EINVAL, "null"),
        (dict(out_dev=None), EINVAL, "null"), (dict(total_dev=None), EINVAL, "null"),
        (dict(form=_native.NORM_FP8, scales_dev=None), EINVAL, "null"), (dict(ldx=99), EINVAL, "stride"), (dict(ldr=99), EINVAL, "stride"),
        (dict(x_dev=SOMEWHERE + 1), ENOTSUP, "aligned"), (dict(residual_dtype=F32, residual_dev=SOMEWHERE + 2), ENOTSUP, "aligned"),
        (dict(weight_dtype=F32, weight_dev=SOMEWHERE + 2), ENOTSUP, "aligned"), (dict(out_dev=SOMEWHERE + 1), ENOTSUP, "aligned"),
        (dict(form=_native.NORM_FP8, out_dev=SOMEWHERE + 4), ENOTSUP, "aligned"), (dict(rstd_dev=SOMEWHERE + 2), ENOTSUP, "aligned"),
    ],
)
def test_norm(fields, status, word):
    assert _native.lib().fsh_rms_norm(_norm(**fields), None) == status
    assert word in _message()


def test_nothing_to_do():
    lib = _native.lib()
    assert lib.fsh_rms_norm(None, None) == EINVAL
    assert lib.fsh_rms_norm(_norm(rows=0, x_dev=None), None) == OK and lib.fsh_rms_norm(_norm(cols=0), None) == OK
    assert lib.fsh_rms_norm_backward(None, None) == EINVAL
    assert lib.fsh_rms_norm_backward(_gradient(rows=0, grad_weight_dev=None), None) == OK
    assert lib.fsh_rms_norm_backward(_gradient(rows=0), None) == ENOTSUP
    assert lib.fsh_act_dequant_1x128(None, None, 0, 5, 128, None, 0, None) == OK
    assert lib.fsh_rms_norm_token_runs(None, 0, 0, 5, 5, None, None, 0, None, 0, None, None) == OK


def _gradient(**fields):
    q = _native.NormGradient()
    for name, kind in q._fields_:
        if kind is ctypes.c_void_p:
            setattr(q, name, SOMEWHERE)
    q.rows, q.cols, q.ldg, q.ldh, q.ldt, q.workspace_nbytes = 4, 100, 100, 100, 100, 1 << 20
    for name, value in fields.items():
        setattr(q, name, value)
    return ctypes.byref(q)


@pytest.mark.parametrize(
    "fields,status,word",
    [
        (dict(rows=-1), EINVAL, "negative"), (dict(grad_dtype=7), EINVAL, "dtype"), (dict(weight_dtype=7), EINVAL, "dtype"),
        (dict(grad_dtype=F32), EINVAL, "gradient of dtype"), (dict(total_dtype=F16), EINVAL, "gradient of dtype"),
        (dict(weight_dev=None), EINVAL, "without a weight"), (dict(grad_dev=None), EINVAL, "null"), (dict(total_dev=None), EINVAL, "null"),
        (dict(rstd_dev=None), EINVAL, "null"), (dict(ldg=99), EINVAL, "stride"), (dict(ldh=99), EINVAL, "stride"), (dict(ldt=99), EINVAL, "stride"),
        (dict(grad_dev=SOMEWHERE + 1), ENOTSUP, "aligned"), (dict(grad_weight_dev=SOMEWHERE + 1), ENOTSUP, "aligned"),
        (dict(rstd_dev=SOMEWHERE + 2), ENOTSUP, "aligned"), (dict(workspace_dev=None), EINVAL, "workspace"),
        (dict(workspace_nbytes=100), EINVAL, "workspace"), (dict(cols=1 << 40, ldg=1 << 40, ldh=1 << 40, ldt=1 << 40, workspace_nbytes=1 << 62), ENOTSUP, "columns"),
    ],
)
def test_gradient(fields, status, word):
    assert _native.lib().fsh_rms_norm_backward(_gradient(**fields), None) == status
    assert word in _message()


def test_workspace_grows_with_neither_beyond_its_groups():
    size = _native.lib().fsh_rms_norm_backward_workspace_bytes
    assert size(0, 5) == size(5, 0) == size(-1, 5) == 0
    assert size(1, 100) == 400 and size(10, 4096) == 10 * 4096 * 4
    assert size(1 << 40, 4096) <= 1024 * 4096 * 4


def test_token_runs_and_dequantize():
    lib = _native.lib()
    args = [SOMEWHERE, BF16, 200, 100, 100, SOMEWHERE, None, 0, SOMEWHERE, 256, SOMEWHERE, None]
    for at, value, status, word in ((1, 5, EINVAL, "dtype"), (2, -1, EINVAL, "negative"), (4, 99, EINVAL, "ldh"), (9, 128, EINVAL, "rounded up"),
                                    (0, None, EINVAL, "null"), (5, None, EINVAL, "null"), (8, SOMEWHERE + 8, ENOTSUP, "aligned"),
                                    (0, SOMEWHERE + 1, ENOTSUP, "aligned"), (2, 1 << 33, EINVAL, "rounded up")):
        assert lib.fsh_rms_norm_token_runs(*args[:at], value, *args[at + 1 :]) == status, (at, value)
        assert word in _message() and _message().startswith("fsh_rms_norm_token_runs")
    huge = [*args]
    huge[2], huge[9] = 128 << 24, 128 << 24
    assert lib.fsh_rms_norm_token_runs(*huge) == ENOTSUP and "tiles" in _message()
    args = [SOMEWHERE, SOMEWHERE, 200, 100, 128, SOMEWHERE, BF16, None]
    for at, value, status, word in ((2, -1, EINVAL, "negative"), (6, 4, EINVAL, "dtype"), (4, 100, EINVAL, "ldq"), (4, 132, ENOTSUP, "aligned"),
                                    (0, None, EINVAL, "null"), (5, SOMEWHERE + 1, ENOTSUP, "aligned")):
        assert lib.fsh_act_dequant_1x128(*args[:at], value, *args[at + 1 :]) == status, (at, value)
        assert word in _message()


def test_there_is_no_cpu_path():
    x = torch.zeros(3, 64)
    for call in (lambda: rms_norm(x), lambda: rms_norm(x.requires_grad_(), torch.ones(64)), lambda: rms_norm_fp8(x), lambda: FlexShardRMSNorm(64)(x)):
        with pytest.raises(RuntimeError, match="CPU"):
            call()
    with pytest.raises(NotImplementedError):
        FlexShardRMSNorm.from_float(torch.nn.RMSNorm((2, 64)))


def test_outputs_that_overlap_inputs():
    far = [SOMEWHERE + (i << 20) for i in range(9)]
    apart = dict(zip(("x_dev", "residual_dev", "weight_dev", "total_dev", "out_dev", "scales_dev", "rstd_dev"), far))
    for fields in (
        dict(out_dev=apart["x_dev"]), dict(total_dev=apart["residual_dev"]), dict(total_dev=apart["x_dev"] + 798),
        dict(out_dev=apart["residual_dev"] + 2 * (3 * 200 + 100) - 2, ldr=200), dict(out_dev=apart["weight_dev"] + 198),
        dict(form=_native.NORM_FP8, out_dev=apart["x_dev"] - 8),
    ):
        assert _native.lib().fsh_rms_norm(_norm(**apart | fields), None) == EINVAL and "overlaps" in _message(), fields
    names = ("grad_dev", "total_dev", "weight_dev", "rstd_dev", "grad_total_dev", "grad_x_dev", "grad_residual_dev", "grad_weight_dev", "workspace_dev")
    apart = dict(zip(names, far))
    for fields in (dict(grad_x_dev=apart["grad_dev"]), dict(grad_x_dev=apart["grad_total_dev"] + 2), dict(grad_x_dev=apart["total_dev"])):
        assert _native.lib().fsh_rms_norm_backward(_gradient(**apart | fields), None) == EINVAL and "overlaps" in _message(), fields


def test_a_norm_under_several_names_is_converted_once():
    """Twice in one parent, and in two: one module under all of its names, as before."""
    norm, other = torch.nn.RMSNorm(8), torch.nn.RMSNorm(8)
    block = torch.nn.ModuleDict({"a": norm, "b": norm, "c": other, "d": torch.nn.Linear(2, 2)})
    model = torch.nn.ModuleList([block, torch.nn.Sequential(norm, other), block])
    model.register_module("nothing", None)
    names = []
    assert convert_to_flex_shard_rms_norm(model, lambda fqn, child: names.append(fqn) or True) is model
    assert type(block["a"]) is FlexShardRMSNorm and block["b"] is block["a"] and model[1][0] is block["a"]
    assert type(block["c"]) is FlexShardRMSNorm and model[1][1] is block["c"] and block["c"] is not block["a"]
    assert block["a"].weight is norm.weight and type(block["d"]) is torch.nn.Linear and model[2] is block
    assert names == ["0.a", "0.b", "0.c", "1.0", "1.1"]


def test_a_name_that_the_filter_leaves_out_keeps_its_norm():
    norm = torch.nn.RMSNorm(8)
    model = torch.nn.ModuleDict({"a": norm, "b": norm, "c": norm})
    convert_to_flex_shard_rms_norm(model, lambda fqn, child: fqn != "b")
    assert type(model["a"]) is FlexShardRMSNorm and model["c"] is model["a"] and model["b"] is norm


def test_outputs_that_overlap_each_other():
    """Or an input that is read late: the factors over a row's end, the scales over the weight, the sum under the norm."""
    lib = _native.lib()
    apart = {name: SOMEWHERE + (i << 20) for i, name in enumerate(("x_dev", "residual_dev", "weight_dev", "total_dev", "out_dev", "scales_dev", "rstd_dev"))}
    fp8 = dict(form=_native.NORM_FP8)
    for fields in (
        dict(out_dev=apart["total_dev"] + 798), dict(total_dev=apart["out_dev"] + 798), fp8 | dict(out_dev=apart["total_dev"] - 504),
        dict(rstd_dev=apart["x_dev"] + 796), dict(rstd_dev=apart["weight_dev"] - 12), dict(rstd_dev=apart["out_dev"]),
        dict(rstd_dev=apart["total_dev"] + 796), fp8 | dict(scales_dev=apart["x_dev"]), fp8 | dict(scales_dev=apart["weight_dev"] - 12),
        fp8 | dict(scales_dev=apart["out_dev"] + 508), fp8 | dict(scales_dev=apart["rstd_dev"] + 12),
    ):
        assert lib.fsh_rms_norm(_norm(**apart | fields), None) == EINVAL and "overlaps" in _message(), fields
    names = ("grad_dev", "total_dev", "weight_dev", "rstd_dev", "grad_total_dev", "grad_x_dev", "grad_residual_dev", "grad_weight_dev", "workspace_dev")
    apart = {name: SOMEWHERE + (i << 20) for i, name in enumerate(names)} | dict(workspace_nbytes=1600)
    wide = dict(total_dtype=F32)
    assert lib.fsh_rms_norm_backward_workspace_bytes(4, 100) == 400  # (what is used of it)
    for fields in (
        dict(grad_x_dev=apart["rstd_dev"] - 796), dict(grad_weight_dev=apart["weight_dev"] + 198), dict(grad_weight_dev=apart["grad_x_dev"] + 798),
        dict(workspace_dev=apart["grad_dev"]), dict(workspace_dev=apart["grad_weight_dev"] - 396), dict(workspace_dev=apart["grad_x_dev"] + 796),
        wide | dict(grad_residual_dev=apart["grad_x_dev"] - 1596), wide | dict(grad_residual_dev=apart["total_dev"] + 1596),
    ):
        assert lib.fsh_rms_norm_backward(_gradient(**apart | fields), None) == EINVAL and "overlaps" in _message(), fields
    h, rstd, weight, q, scales = (SOMEWHERE + (i << 20) for i in range(5))
    for fields in (dict(q=h + 39984), dict(q=rstd - 16), dict(scales=weight), dict(scales=q + 104 * 256 - 4), dict(scales=h)):
        at = dict(q=q, scales=scales) | fields
        assert lib.fsh_rms_norm_token_runs(h, BF16, 200, 100, 100, rstd, weight, BF16, at["q"], 256, at["scales"], None) == EINVAL, fields
        assert "overlaps" in _message()
    for out in (q, q + 199 * 128 + 126, scales + 796):
        assert lib.fsh_act_dequant_1x128(q, scales, 200, 100, 128, out, BF16, None) == EINVAL and "overlaps" in _message()
