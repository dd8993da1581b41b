"""Cases of the operators around a training step's products, each with its plain
form: what is measured of them, and on which sizes.

A case is a dict of plain values; ``op`` says which operator it takes:

``norm``     root-mean-square norm of rows, with the residual's addition or
             without; ``serve`` the outputs alone, ``train`` with the gradients
``norm8``    the same with its output in 8 bits with scales, as the FP8 linear
             multiplies it; returned as the values that it stands for
``squares``  the sum of the squares of many gradients, for clipping by their norm
``adamw``    one AdamW step of many parameters at once, states in 32 or 8 bits,
             the gradients clipped by their norm or as they are

The plain forms compute in 32 bits and round once; ``exact`` computes in 64.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS = 1e-6
RUN = 128  # columns that share a scale of an 8-bit activation
BLOCK = 128  # elements that share a scale of an 8-bit state
MAX_NORM = 1.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
BETAS, ADAM_EPS, DECAY = (0.9, 0.95), 1e-8, 0.1
STEPS_BEFORE = 100  # a run that was resumed


# ------------------------------------------------------------------- the cases
def listed() -> list[dict]:
    return [
        # decoding one sequence: the norm ahead of a layer, nothing but latency
        dict(name="norm_one_token", op="norm", mode="serve", rows=1, cols=4096, dtype="bf16", residual="same", weight="same"),
        # the query heads of 8192 tokens, each normed by itself, in training
        dict(name="norm_heads_train", op="norm", mode="train", rows=8192 * 32, cols=128, dtype="bf16", residual="none", weight="same"),
        # fp32 rows of an odd width, as the small models of the tests have them
        dict(name="norm_odd_rows_train", op="norm", mode="train", rows=1000, cols=1001, dtype="fp32", residual="same", weight="same"),
        # a training step's tokens between two layers
        dict(name="norm_train", op="norm", mode="train", rows=8192, cols=4096, dtype="bf16", residual="same", weight="same"),
        # decoding a batch of sequences into FP8 projections
        dict(name="norm8_48_tokens", op="norm8", mode="serve", rows=48, cols=7168, dtype="bf16", residual="same", weight="same"),
        # a prompt, on an fp32 residual stream
        dict(name="norm8_prompt", op="norm8", mode="serve", rows=8192, cols=7168, dtype="bf16", residual="fp32", weight="fp32"),
        # a training step's tokens into FP8 projections, with the way back
        dict(name="norm8_train", op="norm8", mode="train", rows=8192, cols=4096, dtype="bf16", residual="same", weight="same"),
        # the gradients of a few layers' norm weights, kept in fp32
        dict(name="squares_vectors", op="squares", tensors="vectors", count=20, width=4096, grads="fp32"),
        # the gradients of one Llama-3-8B layer's projections
        dict(name="squares_layer", op="squares", tensors="layer", count=7, width=4096, grads="bf16"),
        # what a Muon step leaves to another optimizer: norm weights, back to back in a bucket, one of an odd size
        dict(name="adamw_vectors", op="adamw", tensors="vectors", count=20, width=4096, params="fp32", grads="fp32", bits=32, clip=True),
        # one Llama-3-8B layer's projections in bf16, fp32 states
        dict(name="adamw_layer", op="adamw", tensors="layer", count=7, width=4096, params="bf16", grads="bf16", bits=32, clip=True),
        # the same as fp32 masters, 8-bit states
        dict(name="adamw8_layer", op="adamw", tensors="layer", count=7, width=4096, params="fp32", grads="fp32", bits=8, clip=False),
    ]


def _spread(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    op = rng.choice(["norm", "norm", "norm8", "norm8", "squares", "adamw", "adamw"])
    if op in ("norm", "norm8"):
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        cols = _spread(rng, 16, 16384)
        rows = min(_spread(rng, 1, 65536), max(1, 8192 * 4096 // cols))
        return dict(op=op, mode=rng.choice(["serve", "train"]), rows=rows, cols=cols, dtype=dtype,
                    residual=rng.choice(["none", "same", "same", "fp32"]), weight=rng.choice(["same", "same", "fp32", "none"]))
    tensors = rng.choice(["vectors", "layer"])
    case = dict(op=op, tensors=tensors, count=rng.randint(1, 20) if tensors == "vectors" else 7,
                width=_spread(rng, 1, 200000) if tensors == "vectors" else _spread(rng, 16, 3000),
                grads=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if op == "adamw":
        bits = rng.choice([32, 8])
        # (8-bit states of fp32 and bf16 parameters; gradients of the parameters' type or of fp32)
        case["params"] = rng.choice(["fp32", "bf16"])
        case["grads"] = rng.choice([case["params"], "fp32"])
        case.update(bits=bits, clip=rng.random() < 0.5)
    return case


def _shapes(case: dict) -> list[tuple[int, ...]]:
    d = case["width"]
    if case["tensors"] == "vectors":
        return [(d + 1,) if i == case["count"] // 2 else (d,) for i in range(case["count"])]
    quarter, wide = max(1, d // 4), 7 * d // 2  # the proportions of a Llama-3-8B layer
    return [(d, d), (quarter, d), (quarter, d), (d, d), (wide, d), (wide, d), (d, wide)]


def work(case: dict) -> dict:
    if case["op"] in ("norm", "norm8"):
        n, e = case["rows"] * case["cols"], SIZE[case["dtype"]]
        stream = 0 if case["residual"] == "none" else 4 if case["residual"] == "fp32" else e
        w = 0 if case["weight"] == "none" else case["cols"] * (4 if case["weight"] == "fp32" else e)
        out = e if case["op"] == "norm" else 1 + 4 / RUN + 2  # 8 bits and scales, and the values in bf16
        total = n * (e + 2 * stream + out) + w
        if case["mode"] == "train":  # the outputs' gradients in, the inputs' out (x and the stream share one of the same type)
            total += n * ((e if case["op"] == "norm" else 2) + stream + e + (stream if stream != e else 0)) + w
        return {"bytes": int(total), "flops": n * (4 if case["mode"] == "serve" else 12)}
    n = sum(math.prod(s) for s in _shapes(case))
    g = SIZE[case["grads"]]
    if case["op"] == "squares":
        return {"bytes": n * g + 8, "flops": 2 * n}
    # 8 bits: the codes of both states in and out, their scales, and the values in bf16
    states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 4
    return {"bytes": int(n * (2 * SIZE[case["params"]] + g + states)), "flops": 15 * n}


# ------------------------------------------------------------------ the inputs
def _generator(seed: int) -> torch.Generator:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _activations(gen, rows: int, cols: int, dtype, scale: float = 1.0) -> torch.Tensor:
    """Normal values with a few channels that stand out, as between a model's layers."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    loud = torch.rand(cols, generator=gen, device="cuda") < 0.01
    x *= torch.where(loud, 12.0 * scale, scale)
    return x.to(dtype)


def _norm_inputs(case: dict, seed: int) -> dict:
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    rows, cols = case["rows"], case["cols"]
    stream = torch.float32 if case["residual"] == "fp32" else dtype
    state = dict(case=case, x=_activations(gen, rows, cols, dtype), residual=None, weight=None)
    if case["residual"] != "none":
        state["residual"] = _activations(gen, rows, cols, stream, 2.0)
    if case["weight"] != "none":
        w = 1.0 + 0.2 * torch.randn(cols, generator=gen, device="cuda")
        state["weight"] = w.to(torch.float32 if case["weight"] == "fp32" else dtype)
    if case["mode"] == "train":
        state["grad"] = _activations(gen, rows, cols, dtype if case["op"] == "norm" else torch.bfloat16, 0.01)
        if state["residual"] is not None:
            state["grad_total"] = _activations(gen, rows, cols, stream, 0.01)
    return state


def _tensor_inputs(case: dict, seed: int) -> dict:
    """Flat buffers that hold the tensors, as a bucket's storage does: back to
    back, or with 8-bit states from multiples of 128 elements on (zeros between)."""
    gen, shapes = _generator(seed), _shapes(case)
    padded = case.get("bits") == 8
    counts = [math.prod(s) for s in shapes]
    slots = [-(-n // BLOCK) * BLOCK if padded else n for n in counts]
    starts = [sum(slots[:i]) for i in range(len(slots))]
    total = sum(slots)

    def zero_gaps(t):
        for start, count, slot in zip(starts, counts, slots):
            t[start + count : start + slot] = 0
        return t

    spread = torch.exp(torch.randn(-(-total // 4096), generator=gen, device="cuda")) * 1e-3
    spread = spread.repeat_interleave(4096)[:total]
    g = zero_gaps(spread * torch.randn(total, generator=gen, device="cuda")).to(DTYPES[case["grads"]])
    state = dict(case=case, shapes=shapes, starts=starts, counts=counts, g=g)
    if case["op"] == "squares":
        return state
    state["p"] = zero_gaps((1.0 if case["tensors"] == "vectors" else 0.0) + 0.02 * torch.randn(total, generator=gen, device="cuda"))
    state["p"] = state["p"].to(DTYPES[case["params"]])
    state["lr"] = 1e-4
    m = zero_gaps(0.3 * spread * torch.randn(total, generator=gen, device="cuda"))
    v = zero_gaps(spread.square() * (0.5 + torch.rand(total, generator=gen, device="cuda")))
    if case["bits"] == 32:
        state.update(m=m, v=v)
        return state
    index = torch.empty(total, dtype=torch.int32, device="cuda")  # of each element in its tensor
    for start, slot in zip(starts, slots):
        index[start : start + slot] = torch.arange(slot, dtype=torch.int32, device="cuda")
    state["index"] = index
    state["m8"], state["m_scale"] = _first_moment_codes(m, index, STEPS_BEFORE)
    state["v8"], state["v_scale"] = _second_moment_codes(v, index, STEPS_BEFORE)
    return state


def _tensors(state: dict, flat: torch.Tensor) -> list[torch.Tensor]:
    """The tensors of a flat buffer, as views."""
    return [flat[s : s + n].view(shape) for s, n, shape in zip(state["starts"], state["counts"], state["shapes"])]


def _inputs(case: dict, seed: int) -> dict:
    return (_norm_inputs if case["op"] in ("norm", "norm8") else _tensor_inputs)(case, seed)


def prepare(case: dict, seed: int) -> dict:
    state = _inputs(case, seed)
    if case["op"] in ("norm", "norm8"):
        if case["mode"] == "train":
            for name in ("x", "residual", "weight"):
                if state[name] is not None:
                    state[name].requires_grad_()
        return state
    state["grads"] = _tensors(state, state["g"])
    state["step"] = STEPS_BEFORE
    if own and case["op"] == "adamw":
        # an optimizer that was resumed from a checkpoint, its gradients in place
        from flex_shard_amd.adamw import FlexShardAdamW

        params = [torch.nn.Parameter(t) for t in _tensors(state, state["p"])]
        optimizer = FlexShardAdamW(params, lr=state["lr"], betas=BETAS, eps=ADAM_EPS, weight_decay=DECAY, state_bits=case["bits"])
        if case["bits"] == 32:
            saved = zip(*[_tensors(state, state[name]) for name in ("m", "v")])
            saved = [dict(step=STEPS_BEFORE, exp_avg=m, exp_avg_sq=v) for m, v in saved]
        else:
            blocks = [(s // BLOCK, -(-(s + n) // BLOCK)) for s, n in zip(state["starts"], state["counts"])]
            saved = [
                dict(step=STEPS_BEFORE, exp_avg=m, exp_avg_scale=state["m_scale"][a:b], exp_avg_sq=v, exp_avg_sq_scale=state["v_scale"][a:b])
                for m, v, (a, b) in zip(_tensors(state, state["m8"]), _tensors(state, state["v8"]), blocks)
            ]
        optimizer.load_state_dict({"state": dict(enumerate(saved)), "param_groups": optimizer.state_dict()["param_groups"]})
        for p, g in zip(params, state["grads"]):
            p.grad_dtype = None
            p.grad = g
        state.update(params=params, optimizer=optimizer)
    return state


# --------------------------------------------------------------------- one pass
def run(state: dict):
    return {"norm": _norm, "norm8": _norm, "squares": _squares, "adamw": _adamw}[state["case"]["op"]](state)


def _norm(state: dict):
    x, residual, weight = state["x"], state["residual"], state["weight"]
    eight, train = state["case"]["op"] == "norm8", state["case"]["mode"] == "train"
    if own:
        from flex_shard_amd.norms import rms_norm, rms_norm_fp8

        with torch.set_grad_enabled(train):
            y = (rms_norm_fp8 if eight else rms_norm)(x, weight, EPS, residual=residual)
            y, total = (y, None) if residual is None else y
            y = y.dequantize(torch.bfloat16) if eight else y
        out = [y.detach()] + ([] if total is None else [total.detach()])
        if not train:
            return out
        wanted = [t for t in (x, residual, weight) if t is not None]
        outputs, grads = ([y], [state["grad"]]) if total is None else ([y, total], [state["grad"], state["grad_total"]])
        return out + list(torch.autograd.grad(outputs, wanted, grads))
    with torch.no_grad():
        h = x.float()
        if residual is not None:
            total = (h + residual.float()).to(residual.dtype)
            h = total.float()
        s = 1.0 / torch.sqrt((h * h).mean(dim=-1, keepdim=True) + EPS)
        y = h * s if weight is None else h * s * weight.float()
        y = _through_8_bits(y.to(torch.bfloat16).float()).to(torch.bfloat16) if eight else y.to(x.dtype)
        out = [y] if residual is None else [y, total]
        if not train:
            return out
        g = state["grad"].float()
        a = g if weight is None else g * weight.float()
        n = h * s
        grad = s * (a - n * (a * n).mean(dim=-1, keepdim=True))
        if residual is None:
            out.append(grad.to(x.dtype))
        else:
            grad = grad + state["grad_total"].float()
            out += [grad.to(x.dtype), grad.to(residual.dtype)]
        return out if weight is None else out + [(g * n).sum(dim=0).to(weight.dtype)]


def _squares(state: dict):
    if own:
        from flex_shard_amd.adamw import grad_square_sum

        return grad_square_sum(state["grads"])
    return state["g"].double().square().sum()  # (a long sum)


def _adamw(state: dict):
    case, clip, eight = state["case"], state["case"]["clip"], state["case"]["bits"] == 8
    if own:
        from flex_shard_amd.adamw import grad_square_sum

        optimizer, params = state["optimizer"], state["params"]
        if clip:
            optimizer.step(square_sum=grad_square_sum(state["grads"]), max_norm=MAX_NORM)
        else:
            optimizer.step()
        if eight:
            states = [optimizer.state_values(p, torch.bfloat16) for p in params]
        else:
            states = [(optimizer.state[p]["exp_avg"], optimizer.state[p]["exp_avg_sq"]) for p in params]
        return [p.detach() for p in params], [m for m, _ in states], [v for _, v in states]
    with torch.no_grad():
        state["step"] = t = state["step"] + 1
        g, p = state["g"].float(), state["p"].float()
        if clip:
            norm = state["g"].double().square().sum().sqrt()
            g = g * (MAX_NORM / (norm + 1e-6)).clamp(max=1.0).float()
        if eight:
            m = _first_moment_values(state["m8"], state["m_scale"])
            v = _second_moment_values(state["v8"], state["v_scale"])
        else:
            m, v = state["m"], state["v"]
        (b1, b2), lr = BETAS, state["lr"]
        m = m * b1 + g * (1 - b1)
        v = v * b2 + (g * g) * (1 - b2)
        root = torch.sqrt(v) * (1.0 / math.sqrt(1 - b2**t)) + ADAM_EPS
        p = p * (1 - lr * DECAY) - (lr / (1 - b1**t)) * (m / root)
        state["p"].copy_(p.to(state["p"].dtype))
        if eight:
            state["m8"], state["m_scale"] = _first_moment_codes(m, state["index"], t)
            state["v8"], state["v_scale"] = _second_moment_codes(v, state["index"], t)
            m = _first_moment_values(state["m8"], state["m_scale"]).to(torch.bfloat16)
            v = _second_moment_values(state["v8"], state["v_scale"]).to(torch.bfloat16)
        else:
            state["m"], state["v"] = m, v
        return _tensors(state, state["p"]), _tensors(state, m), _tensors(state, v)


# ----------------------------------------------------------------- plain pieces
def _through_8_bits(y: torch.Tensor) -> torch.Tensor:
    """fp32 rows to E4M3 with a scale for every run of 128 columns, and back:
    448 over the run's largest magnitude (at least 1e-12) takes it to E4M3's."""
    cols = y.shape[-1]
    runs = torch.nn.functional.pad(y, (0, -cols % RUN)).unflatten(-1, (-1, RUN))
    scale = (448.0 / runs.abs().amax(dim=-1, keepdim=True).clamp(min=1e-12).double()).float()
    values = (runs * scale).to(torch.float8_e4m3fn).float() * (1.0 / scale)
    return values.flatten(-2)[..., :cols]


# Eight-bit states: 128 elements share a scale, their largest magnitude (at least
# 2**-100).  A code stands for the fp32 number whose upper bits, 3 of the mantissa
# and those of the exponent, it counts down from 1.0 = 1016 * 2**20: the first
# moment has a sign and the codes 1 to 127 (to 1.0), the second the codes 1 to 255; 0
# is zero.  Rounding up or down goes by a dither in [0, 1) that every element has anew
# in every step: half of a word that is mixed from the element's index and the step's.
def _dither(index: torch.Tensor, t: int) -> torch.Tensor:
    z = (index.long() * 0x9E3779B9 + t * 0x6A09E667) & 0xFFFFFFFF
    z = ((z ^ (z >> 16)) * 0xBB67AE85) & 0xFFFFFFFF
    return z ^ (z >> 15)


def _scaled(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    blocks = x.view(-1, BLOCK)
    scale = blocks.abs().amax(dim=-1, keepdim=True).clamp(min=2.0**-100)
    return (blocks.abs() * (torch.ones_like(scale) / scale)).clamp(max=1.0).view(-1), scale.view(-1)


def _first_moment_codes(m: torch.Tensor, index: torch.Tensor, t: int) -> tuple[torch.Tensor, torch.Tensor]:
    size, scale = _scaled(m)
    u = (_dither(index, t) & 0xFFFF) << 16
    code = ((size.view(torch.int32) + (u >> 12)) >> 20) - 889
    smallest = 1.25 * 2.0**-16
    few = (size * (1.0 / smallest) > (u >> 8).float() * 2.0**-24).long()
    code = torch.where(size < smallest, few, code)
    return (code | torch.where(m < 0, 128, 0)).to(torch.uint8), scale


def _second_moment_codes(v: torch.Tensor, index: torch.Tensor, t: int) -> tuple[torch.Tensor, torch.Tensor]:
    size, scale = _scaled(v)
    u = _dither(index, t) >> 16 << 16
    code = ((size.view(torch.int32) + (u >> 12)) >> 20) - 761
    # (what is not zero stays so: a first moment is never divided by nothing)
    return torch.where(size > 0, code.clamp(min=1), 0).to(torch.uint8), scale


def _first_moment_values(code: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    size = (code & 127).int()
    value = torch.where(size > 0, (size + 889) << 20, 0).view(torch.float32)
    value = torch.where(code > 127, -value, value)
    return (value.view(-1, BLOCK) * scale[:, None]).view(-1)


def _second_moment_values(code: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    value = torch.where(code > 0, (code.int() + 761) << 20, 0).view(torch.float32)
    return (value.view(-1, BLOCK) * scale[:, None]).view(-1)


# ---------------------------------------------------------------- in 64 bits
def exact(case: dict, seed: int):
    state = _inputs(case, seed)
    return {"norm": _exact_norm, "norm8": _exact_norm, "squares": _exact_squares, "adamw": _exact_adamw}[case["op"]](state)


def _exact_norm(state: dict):
    case, residual, weight = state["case"], state["residual"], state["weight"]
    h = state["x"].double()
    out = []
    if residual is not None:
        out = [h + residual.double()]
        h = out[0].to(residual.dtype).double()  # the stream is kept in its type
    cols = case["cols"]
    root = torch.sqrt(torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / cols + EPS)
    w = 1.0 if weight is None else weight.double()
    y = h / root * w
    if case["op"] == "norm8":
        y = _exact_8_bits(y.to(torch.bfloat16).double())
    out = [y, *out]
    if case["mode"] == "serve":
        return out
    g = state["grad"].double()
    # y_j = w_j h_j / root, d root / d h_i = h_i / (cols root)
    along = (g * w * h).sum(dim=1, keepdim=True)
    grad = g * w / root - h * along / (cols * root**3)
    if residual is not None:
        grad = grad + state["grad_total"].double()
    out += [grad] if residual is None else [grad, grad]
    return out if weight is None else [*out, (g * h / root).sum(dim=0)]


def _exact_8_bits(y: torch.Tensor) -> torch.Tensor:
    """Runs of 128 columns over their scale, to the nearest multiple of an E4M3
    step: 2**-3 of the power of two below, 2**-9 under 2**-6."""
    rows, cols = y.shape
    runs = torch.zeros(rows, -(-cols // RUN), RUN, dtype=torch.float64, device=y.device)
    runs.view(rows, -1)[:, :cols] = y
    scale = torch.maximum(runs.abs().max(dim=-1, keepdim=True).values, torch.tensor(1e-12, device=y.device).double()) / 448.0
    v = runs / scale
    _, exponent = torch.frexp(v)
    step = torch.exp2((exponent - 4).clamp(min=-9).double())
    return (torch.round(v / step) * step * scale).view(rows, -1)[:, :cols].clone()


def _exact_squares(state: dict):
    return sum(np.float64(t.double().square().sum().item()) for t in _tensors(state, state["g"]))


def _exact_adamw(state: dict):
    case, t, (b1, b2), lr = state["case"], STEPS_BEFORE + 1, BETAS, state["lr"]
    eight = case["bits"] == 8
    factor = 1.0
    if case["clip"]:
        factor = min(1.0, MAX_NORM / (math.sqrt(_exact_squares(state)) + 1e-6))
    params, firsts, seconds = [], [], []
    for start, count, shape in zip(state["starts"], state["counts"], state["shapes"]):
        part = slice(start, start + count)
        p, g = state["p"][part].double(), state["g"][part].double() * factor
        if eight:
            part = slice(start // BLOCK, -(-(start + count) // BLOCK))
            codes = [state[name].view(-1, BLOCK)[part].long() for name in ("m8", "v8")]
            size = codes[0] % 128
            m = torch.where(size > 0, _at(size - 127), 0.0) * torch.where(codes[0] >= 128, -1.0, 1.0) * state["m_scale"][part, None].double()
            v = torch.where(codes[1] > 0, _at(codes[1] - 255), 0.0) * state["v_scale"][part, None].double()
            m, v = m.view(-1)[:count], v.view(-1)[:count]
        else:
            m, v = state["m"][part].double(), state["v"][part].double()
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g**2
        p = p - lr * DECAY * p - lr * (m / (1 - b1**t)) / (torch.sqrt(v / (1 - b2**t)) + ADAM_EPS)
        if eight:
            m, v = _exact_state(m, t, 127), _exact_state(v, t, 255)
        for kept, value in zip((params, firsts, seconds), (p, m, v)):
            kept.append(value.view(shape))
    return params, firsts, seconds


def _at(place: torch.Tensor) -> torch.Tensor:
    """The numbers of 3 mantissa bits in their order, 1.0 at place 0."""
    octave = torch.div(place, 8, rounding_mode="floor")
    return (1.0 + (place - 8 * octave) / 8.0) * torch.exp2(octave.double())


def _exact_state(x: torch.Tensor, t: int, codes: int) -> torch.Tensor:
    """Up to the next of the numbers of a code where the dither is less than what
    is missing of the step above it, down otherwise."""
    count = x.numel()
    blocks = torch.zeros(-(-count // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    blocks[:count] = x
    blocks = blocks.view(-1, BLOCK)
    scale = blocks.abs().max(dim=1, keepdim=True).values.clamp(min=2.0**-100)
    size = blocks.abs() / scale
    index = torch.arange(blocks.numel(), device=x.device).view_as(blocks)
    word = (index * 0x9E3779B9 + t * 0x6A09E667) % 2**32
    word = (word ^ word // 2**16) * 0xBB67AE85 % 2**32
    word = word ^ word // 2**15
    u = (word % 2**16 if codes == 127 else word // 2**16).double() / 2**16
    _, exponent = torch.frexp(size)
    step = torch.exp2((exponent - 4).double())
    below = torch.floor(size / step)
    value = torch.where(size / step - below + u >= 1.0, below + 1.0, below) * step
    smallest = 1.25 * (2.0**-16 if codes == 127 else 2.0**-32)
    if codes == 127:
        value = torch.where(size < smallest, torch.where(size / smallest > u, smallest, 0.0), value)
    else:
        value = torch.where(size > 0, value.clamp(min=smallest), 0.0)
    return (torch.sign(blocks) * value * scale).view(-1)[:count]
