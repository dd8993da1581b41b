"""Cases of the operators for 4-bit training and serving and for experts, each
with its plain form: what is measured of them, and on which sizes.

A case is a dict of plain values; ``op`` says which operator it takes:

``quantize``  a matrix to microscaled 4-bit floats (E2M1 elements, one power
              of two for 32 of them) and back to the values they stand for;
              ``form``: runs along its rows, along its columns, or both
``linear``    a linear layer on operands quantized that way: ``serve`` with a
              weight that was quantized once, ``train`` on a weight that changes
              from step to step, with the gradients
``tokens``    tokens sorted by expert and gathered, and the experts' rows
              brought back with the router's weights; ``train`` with gradients
``experts``   every expert's linear layer on its own tokens, ``serve`` or
              ``train`` as above

The plain forms compute in 32 bits and round once; ``exact`` computes in 64.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = 32  # elements that share a scale
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------- the cases
def listed() -> list[dict]:
    return [
        # one token's activation on its way into a 4-bit product: nothing but latency
        dict(name="quantize_one_token", op="quantize", rows=1, cols=4096, dtype="bf16", form="rows"),
        # 8192 tokens of a training step, for the layer's product and for its weight gradient
        dict(name="quantize_activations_both_ways", op="quantize", rows=8192, cols=4096, dtype="bf16", form="both"),
        # the fp32 master of a gate projection
        dict(name="quantize_master_weight", op="quantize", rows=14336, cols=4096, dtype="fp32", form="both"),
        # decoding one sequence: the gate projection of a Llama-3-8B layer, bound by the weight's bytes
        dict(name="linear_one_token", op="linear", mode="serve", tokens=1, n=14336, k=4096, dtype="bf16", bias=True),
        # decoding a batch of sequences
        dict(name="linear_48_tokens", op="linear", mode="serve", tokens=48, n=14336, k=4096, dtype="bf16", bias=False),
        # a prompt of a length that fits no tile, in fp16, with a bias
        dict(name="linear_ragged_prompt", op="linear", mode="serve", tokens=1000, n=5120, k=2048, dtype="fp16", bias=True),
        # a training step of the gate projection
        dict(name="linear_train", op="linear", mode="train", tokens=8192, n=14336, k=4096, dtype="bf16", bias=True),
        # decoding 16 sequences: where their tokens go, and what comes back
        dict(name="tokens_decode", op="tokens", mode="serve", tokens=16, top_k=8, experts=32, width=7168, dtype="bf16", absent=0.0),
        # a few odd-sized fp32 rows over few experts, a third of the choices at experts of other ranks
        dict(name="tokens_odd_rows", op="tokens", mode="train", tokens=1000, top_k=2, experts=5, width=1001, dtype="fp32", absent=0.3),
        # a training step's tokens
        dict(name="tokens_train", op="tokens", mode="train", tokens=8192, top_k=8, experts=32, width=7168, dtype="bf16", absent=0.0),
        # decoding 16 sequences: the up projections of one rank's DeepSeek-V3 experts, a few tokens each
        dict(name="experts_decode", op="experts", mode="serve", tokens=16, top_k=8, experts=32, n=2048, k=7168, dtype="bf16",
             absent=0.0, sorted=False),
        # a training step of them
        dict(name="experts_train", op="experts", mode="train", tokens=4096, top_k=8, experts=32, n=2048, k=7168, dtype="bf16",
             absent=0.05, sorted=False),
    ]


def _spread(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    op = rng.choice(["quantize", "linear", "tokens", "experts"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "quantize":
        rows, cols = _spread(rng, 1, 16384), _spread(rng, 32, 14336)
        while rows * cols > 8192 * 7168:
            rows = max(1, rows // 2)
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, form=rng.choice(["rows", "columns", "both"]))
    if op == "linear":
        mode = rng.choice(["serve", "serve", "train"])
        case = dict(op=op, mode=mode, tokens=_spread(rng, 1, 8192), n=_spread(rng, 64, 14336), k=_spread(rng, 64, 14336),
                    dtype=dtype, bias=rng.random() < 0.5)
        while case["tokens"] * case["n"] * case["k"] > 8192 * 4096 * 4096:
            case["tokens"] = max(1, case["tokens"] // 2)
            case["n"] = max(64, case["n"] // 2) if case["tokens"] == 1 else case["n"]
        return case
    experts = rng.choice([1, 5, 8, 32, 64, 256]) if op == "tokens" else rng.choice([1, 4, 8, 32])
    top_k = rng.randint(1, min(8, experts))
    mode, absent = rng.choice(["serve", "train"]), rng.choice([0.0, 0.0, 0.1, 0.5])
    if op == "tokens":
        case = dict(op=op, mode=mode, tokens=_spread(rng, 1, 8192), top_k=top_k, experts=experts, width=_spread(rng, 64, 7168),
                    dtype=dtype, absent=absent)
        while case["tokens"] * top_k * case["width"] > 8192 * 8 * 4096:
            case["tokens"] = max(1, case["tokens"] // 2)
        return case
    case = dict(op=op, mode=mode, tokens=_spread(rng, 1, 4096), top_k=top_k, experts=experts, n=_spread(rng, 64, 4096),
                k=_spread(rng, 64, 7168), dtype=dtype, absent=absent, sorted=rng.random() < 0.5)
    while case["tokens"] * top_k * case["n"] * case["k"] > 16384 * 2048 * 7168 or experts * case["n"] * case["k"] > 32 * 2048 * 4096:
        case["tokens"] = max(1, case["tokens"] // 2)
        case["n"] = max(64, case["n"] * 3 // 4)
    return case


def work(case: dict) -> dict:
    e = SIZE[case["dtype"]]
    four = 0.5 + 1.0 / BLOCK  # bytes that an element and its part of a scale take
    if case["op"] == "quantize":
        count = case["rows"] * case["cols"]
        forms = 2 if case["form"] == "both" else 1
        return {"bytes": int(count * (e + forms * (four + e))), "flops": 0}
    if case["op"] == "linear":
        m, n, k = case["tokens"], case["n"], case["k"]
        bias = n * e if case["bias"] else 0
        if case["mode"] == "serve":
            return {"bytes": int(m * k * e + n * k * four + bias + m * n * e), "flops": 2 * m * n * k}
        return {"bytes": 2 * (m * k + n * k + m * n) * e + 2 * bias, "flops": 6 * m * n * k}
    m = case["tokens"] * case["top_k"]
    here = int(round(m * (1.0 - case["absent"])))  # rows that experts of this rank get
    if case["op"] == "tokens":
        t, d = case["tokens"], case["width"]
        ids = m * 8
        forward = t * d * e + m * d * e + ids + m * 4 + here * d * e + m * 4 + t * d * e
        if case["mode"] == "serve":
            return {"bytes": forward, "flops": 2 * here * d}
        # the gradients of the gathered tokens, of the experts' rows and of the weights
        return {"bytes": forward + here * d * e + t * d * e + t * d * e + m * d * e + m * 4, "flops": 7 * here * d}
    n, k, count = case["n"], case["k"], case["experts"]
    rows_in = (m if case["sorted"] else case["tokens"]) * k
    if case["mode"] == "serve":
        hit = count * (1.0 - (1.0 - (1.0 - case["absent"]) * case["top_k"] / count) ** case["tokens"])  # experts with a token
        return {"bytes": int(rows_in * e + m * 8 + hit * n * k * four + m * n * e), "flops": 2 * here * n * k}
    return {"bytes": 2 * rows_in * e + m * 8 + 2 * count * n * k * e + 2 * m * n * e, "flops": 6 * here * n * k}


# ------------------------------------------------------------------ the inputs
def _generator(case: dict, seed: int) -> torch.Generator:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _activations(gen, rows: int, cols: int, dtype, scale: float = 1.0) -> torch.Tensor:
    """Normal values with a few channels that stand out, as between a model's layers."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    loud = torch.rand(cols, generator=gen, device="cuda") < 0.01
    x *= torch.where(loud, 12.0 * scale, scale)
    return x.to(dtype)


def _weights(gen, shape, dtype) -> torch.Tensor:
    return (torch.randn(*shape, generator=gen, device="cuda") * 0.02).to(dtype)


def _choices(gen, case: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """What a router hands on: per token the experts of its ``top_k`` largest
    probabilities (some experts are liked better), and those probabilities; a
    choice whose expert lives on another rank is -1."""
    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    logits = torch.randn(tokens, experts, generator=gen, device="cuda")
    logits += 0.5 * torch.randn(experts, generator=gen, device="cuda")
    weights, ids = torch.softmax(logits, dim=-1).topk(top_k, dim=-1)
    away = torch.rand(tokens, top_k, generator=gen, device="cuda") < case["absent"]
    return torch.where(away, -1, ids), weights.contiguous()


def prepare(case: dict, seed: int) -> dict:
    state = _inputs(case, seed)
    if case["op"] in ("linear", "experts") and case["mode"] == "serve":
        # a server quantizes its weights once
        if own:
            from flex_shard_amd.mxfp4 import quantize_mxfp4_weight

            state["weight"] = quantize_mxfp4_weight(state["weight"])
        else:
            state["weight"] = _through_4_bits(state["weight"].float())
    if case["op"] in ("linear", "experts") and case["mode"] == "train":
        state["x"].requires_grad_()
        state["weight"].requires_grad_()
        if state.get("bias") is not None:
            state["bias"].requires_grad_()
    if case["op"] == "tokens" and case["mode"] == "train":
        for name in ("x", "rows", "weights"):
            state[name].requires_grad_()
    return state


def _inputs(case: dict, seed: int) -> dict:
    gen, dtype = _generator(case, seed), DTYPES[case["dtype"]]
    if case["op"] == "quantize":
        return dict(case=case, x=_activations(gen, case["rows"], case["cols"], dtype))
    if case["op"] == "linear":
        state = dict(case=case, x=_activations(gen, case["tokens"], case["k"], dtype),
                     weight=_weights(gen, (case["n"], case["k"]), dtype),
                     bias=_weights(gen, (case["n"],), dtype) if case["bias"] else None)
        if case["mode"] == "train":
            state["grad"] = _activations(gen, case["tokens"], case["n"], dtype, 0.01)
        return state
    ids, weights = _choices(gen, case)
    m = case["tokens"] * case["top_k"]
    if case["op"] == "tokens":
        width = case["width"]
        state = dict(case=case, ids=ids, weights=weights, x=_activations(gen, case["tokens"], width, dtype),
                     rows=_activations(gen, m, width, dtype))
        if case["mode"] == "train":
            state["grad_sorted"] = _activations(gen, m, width, dtype, 0.01)
            state["grad"] = _activations(gen, case["tokens"], width, dtype, 0.01)
        return state
    state = dict(case=case, ids=ids, x=_activations(gen, m if case["sorted"] else case["tokens"], case["k"], dtype),
                 weight=_weights(gen, (case["experts"], case["n"], case["k"]), dtype))
    if case["mode"] == "train":
        state["grad"] = _activations(gen, m, case["n"], dtype, 0.01)
    return state


# --------------------------------------------------------------------- one pass
def run(state: dict):
    op = {"quantize": _quantize, "linear": _linear, "tokens": _tokens, "experts": _experts}[state["case"]["op"]]
    return op(state)


def _quantize(state: dict):
    x, form = state["x"], state["case"]["form"]
    if own:
        from flex_shard_amd.mxfp4 import mxfp4_quantize, mxfp4_quantize_both, mxfp4_quantize_transposed

        if form == "both":
            return tuple(matrix.dequantize(x.dtype) for matrix in mxfp4_quantize_both(x))
        return (mxfp4_quantize(x) if form == "rows" else mxfp4_quantize_transposed(x)).dequantize(x.dtype)
    rows = None if form == "columns" else _through_4_bits(x.float()).to(x.dtype)
    columns = None if form == "rows" else _through_4_bits(x.float().t().contiguous()).to(x.dtype)
    return (rows, columns) if form == "both" else rows if form == "rows" else columns


def _linear(state: dict):
    x, weight, bias = state["x"], state["weight"], state["bias"]
    train = state["case"]["mode"] == "train"
    if own:
        from flex_shard_amd.mxfp4 import mxfp4_linear

        if not train:
            with torch.no_grad():
                return mxfp4_linear(x, weight, bias)
        y = mxfp4_linear(x, weight, bias)
        wanted = (x, weight) if bias is None else (x, weight, bias)
        return (y.detach(), *torch.autograd.grad(y, wanted, state["grad"]))
    with torch.no_grad():
        x32 = x.float()
        w = _through_4_bits(weight.float()) if train else weight
        y = _through_4_bits(x32) @ w.t()
        if bias is not None:
            y = y + bias.float()
        y = y.to(x.dtype)
        if not train:
            return y
        g = state["grad"].float()
        gx = _through_4_bits(g) @ _through_4_bits(weight.float().t().contiguous()).t()
        gw = _through_4_bits(g.t().contiguous()) @ _through_4_bits(x32.t().contiguous()).t()
        out = (y, gx.to(x.dtype), gw.to(weight.dtype))
        return out if bias is None else (*out, g.sum(dim=0).to(bias.dtype))


def _tokens(state: dict):
    case, ids, x, rows, weights = state["case"], state["ids"], state["x"], state["rows"], state["weights"]
    train = case["mode"] == "train"
    if own:
        from flex_shard_amd.experts import combine_tokens, dispatch_tokens, route_tokens

        with torch.set_grad_enabled(train):
            routing = route_tokens(ids, case["experts"])
            gathered = dispatch_tokens(x, routing)
            back = combine_tokens(rows, routing, weights)
        out = (routing.position, routing.offsets, gathered.detach(), back.detach())
        if not train:
            return out
        (grad_x,) = torch.autograd.grad(gathered, x, state["grad_sorted"])
        return (*out, grad_x, *torch.autograd.grad(back, (rows, weights), state["grad"]))
    with torch.no_grad():
        position, offsets, source, here = _sorted_choices(ids, case["experts"])
        m, top_k = source.numel(), case["top_k"]
        of_row = torch.where(here, source // top_k, 0)
        gathered = torch.where(here[:, None], x.float()[of_row], 0.0).to(x.dtype)
        at, taken = position.clamp(min=0).long(), (position >= 0)[..., None]
        back = (torch.where(taken, rows.float()[at], 0.0) * weights.float()[..., None]).sum(dim=1).to(x.dtype)
        out = (position.int(), offsets.int(), gathered, back)
        if not train:
            return out
        grad_x = torch.where(taken, state["grad_sorted"].float()[at], 0.0).sum(dim=1).to(x.dtype)
        g = state["grad"].float()
        w_of_row = weights.float().reshape(-1)[torch.where(here, source, 0)]
        grad_rows = torch.where(here[:, None], w_of_row[:, None] * g[of_row], 0.0).to(x.dtype)
        grad_weights = torch.where(taken, rows.float()[at] * g[:, None, :], 0.0).sum(dim=-1).to(weights.dtype)
        return (*out, grad_x, grad_rows, grad_weights)


def _experts(state: dict):
    case, ids, x, weight = state["case"], state["ids"], state["x"], state["weight"]
    train = case["mode"] == "train"
    if own:
        from flex_shard_amd.experts import route_tokens
        from flex_shard_amd.mxfp4 import mxfp4_expert_linear

        routing = route_tokens(ids, case["experts"])
        if not train:
            with torch.no_grad():
                return mxfp4_expert_linear(x, weight, routing, sorted_rows=case["sorted"])
        y = mxfp4_expert_linear(x, weight, routing, sorted_rows=case["sorted"])
        return (y.detach(), *torch.autograd.grad(y, (x, weight), state["grad"]))
    with torch.no_grad():
        position, offsets, source, here = _sorted_choices(ids, case["experts"])
        of_row = torch.where(here, source // case["top_k"], 0)
        x32 = x.float()
        x4 = _through_4_bits(x32)
        m, n, k = source.numel(), case["n"], case["k"]
        y = torch.zeros(m, n, device=x.device)
        if train:
            g = state["grad"].float()
            g4 = _through_4_bits(g)
            gx_sorted = torch.zeros(m, k, device=x.device)
            gw = torch.zeros(case["experts"], n, k, device=x.device)
        ends = offsets.tolist()
        for e in range(case["experts"]):
            begin, end = ends[e], ends[e + 1]
            if begin == end:
                continue
            part = slice(begin, end) if case["sorted"] else of_row[begin:end]
            w = _through_4_bits(weight[e].float()) if train else weight[e]
            y[begin:end] = x4[part] @ w.t()
            if train:
                gx_sorted[begin:end] = g4[begin:end] @ _through_4_bits(weight[e].float().t().contiguous()).t()
                over_tokens = _through_4_bits(g[begin:end].t().contiguous())
                gw[e] = over_tokens @ _through_4_bits(x32[part].t().contiguous()).t()
        y = y.to(x.dtype)
        if not train:
            return y
        if case["sorted"]:
            gx = gx_sorted
        else:
            gx = torch.where((position >= 0)[..., None], gx_sorted[position.clamp(min=0).long()], 0.0).sum(dim=1)
        return y, gx.to(x.dtype), gw.to(weight.dtype)


# ----------------------------------------------------------------- plain pieces
def _through_4_bits(x: torch.Tensor) -> torch.Tensor:
    """fp32 rows to microscaled 4-bit floats and back: of every run of 32 the
    scale is the power of two of its largest magnitude, less 2 (the largest
    element is 6 = 1.5 * 2**2), the elements round to nearest even among 0, 0.5,
    1, 1.5, 2, 3, 4, 6 and stop at 6."""
    cols = x.shape[-1]
    runs = torch.nn.functional.pad(x, (0, -cols % BLOCK)).unflatten(-1, (-1, BLOCK))
    _, exponent = torch.frexp(runs.abs().amax(dim=-1, keepdim=True))
    scale = torch.ldexp(torch.ones_like(runs[..., :1]), (exponent - 3).clamp(min=-126))
    v = runs / scale
    size = v.abs()
    step = torch.where(size < 2.0, 0.5, torch.where(size < 4.0, 1.0, 2.0))
    v = torch.copysign((torch.round(size / step) * step).clamp(max=6.0), v)
    return (v * scale).flatten(-2)[..., :cols]


def _sorted_choices(ids: torch.Tensor, experts: int):
    """The stable order of the choices by expert, those at no expert of this
    rank last: the sorted row of each choice (-1: none), the first row of each
    expert, the choice of each row, and whether the row is used."""
    flat = ids.reshape(-1)
    key = torch.where((flat < 0) | (flat >= experts), experts, flat)
    source = torch.argsort(key, stable=True)
    position = torch.empty_like(source)
    position[source] = torch.arange(source.numel(), device=ids.device)
    counts = (key[:, None] == torch.arange(experts, device=ids.device)).sum(dim=0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    here = torch.arange(source.numel(), device=ids.device) < offsets[-1]
    position = torch.where(key < experts, position, -1).view(ids.shape)
    return position, offsets, source, here


# ---------------------------------------------------------------- in 64 bits
_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_4_bits(x: torch.Tensor) -> torch.Tensor:
    """What float64 rows stand for in 4 bits, from the definition: the nearest
    of the eight magnitudes by their distances, the one with the even code where
    two are equally near."""
    rows, cols = x.shape
    out = torch.zeros(rows, -(-cols // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    out[:, :cols] = x
    runs = out.view(rows, -1, BLOCK)
    largest = runs.abs().amax(dim=-1)
    power = torch.where(largest > 0, torch.floor(torch.log2(torch.where(largest > 0, largest, 1.0))), -125.0)
    # (a logarithm may round up to the next whole number, or down from one)
    power = torch.where(torch.exp2(power) > largest, power - 1, power)
    power = torch.where(torch.exp2(power + 1) <= largest, power + 1, power)
    scale = torch.exp2((power - 2).clamp(min=-127.0))[..., None]
    wanted = runs.abs() / scale
    best = torch.zeros_like(wanted)
    for code in range(1, 8):
        below, value = _VALUES[code - 1], _VALUES[code]
        nearer = (value - wanted) < (wanted - below)
        even = ((value - wanted) == (wanted - below)) & (code % 2 == 0)
        best = torch.where(nearer | even, value, best)
    return (torch.sign(runs) * best * scale).view(rows, -1)[:, :cols]


def exact(case: dict, seed: int):
    state = _inputs(case, seed)
    return {"quantize": _exact_quantize, "linear": _exact_linear, "tokens": _exact_tokens, "experts": _exact_experts}[case["op"]](state)


def _exact_quantize(state: dict):
    x, form = state["x"].double(), state["case"]["form"]
    if form == "rows":
        return _exact_4_bits(x)
    columns = _exact_4_bits(x.t().contiguous())
    return columns if form == "columns" else (_exact_4_bits(x), columns)


def _exact_linear(state: dict):
    x, w = state["x"].double(), state["weight"].double()
    y = torch.mm(_exact_4_bits(x), _exact_4_bits(w).t())
    if state["bias"] is not None:
        y += state["bias"].double()
    if state["case"]["mode"] == "serve":
        return y
    g = state["grad"].double()
    gx = torch.mm(_exact_4_bits(g), _exact_4_bits(w.t().contiguous()).t())
    gw = torch.mm(_exact_4_bits(g.t().contiguous()), _exact_4_bits(x.t().contiguous()).t())
    return (y, gx, gw) if state["bias"] is None else (y, gx, gw, g.sum(dim=0))


def _exact_order(ids: torch.Tensor, experts: int):
    """On the host, by counting: per expert the flat numbers of its choices."""
    flat = ids.reshape(-1).cpu().numpy()
    chosen = [np.flatnonzero(flat == e) for e in range(experts)]
    offsets = np.concatenate([[0], np.cumsum([len(c) for c in chosen])])
    position = np.full(flat.shape, -1, dtype=np.int64)
    for e in range(experts):
        position[chosen[e]] = offsets[e] + np.arange(len(chosen[e]))
    return chosen, offsets, position


def _exact_tokens(state: dict):
    case, device = state["case"], state["x"].device
    chosen, offsets, position = _exact_order(state["ids"], case["experts"])
    source = torch.from_numpy(np.concatenate(chosen)).to(device)
    used, top_k = source.numel(), case["top_k"]
    token, x, rows, weights = source // top_k, state["x"].double(), state["rows"], state["weights"].double().reshape(-1)
    gathered = torch.zeros(rows.shape, dtype=torch.float64, device=device)
    gathered[:used] = x[token]
    back = torch.zeros_like(x)
    back.index_add_(0, token, rows[:used].double() * weights[source, None])
    out = (torch.from_numpy(position).view(state["ids"].shape).to(device).int(), torch.from_numpy(offsets).to(device).int(), gathered, back)
    if case["mode"] == "serve":
        return out
    grad_x = torch.zeros_like(x)
    grad_x.index_add_(0, token, state["grad_sorted"][:used].double())
    g = state["grad"].double()
    grad_rows = torch.zeros(rows.shape, dtype=torch.float64, device=device)
    grad_rows[:used] = g[token] * weights[source, None]
    grad_weights = torch.zeros_like(weights)
    grad_weights[source] = (g[token] * rows[:used].double()).sum(dim=1)
    return (*out, grad_x, grad_rows, grad_weights.view(state["weights"].shape))


def _exact_experts(state: dict):
    case, device = state["case"], state["x"].device
    chosen, offsets, _ = _exact_order(state["ids"], case["experts"])
    train, m = case["mode"] == "train", state["ids"].numel()
    y = torch.zeros(m, case["n"], dtype=torch.float64, device=device)
    gx = torch.zeros(state["x"].shape, dtype=torch.float64, device=device)
    gw = torch.zeros(state["weight"].shape, dtype=torch.float64, device=device) if train else None
    for e, choices in enumerate(chosen):
        begin, end = int(offsets[e]), int(offsets[e + 1])
        if begin == end:
            continue
        rows = torch.arange(begin, end, device=device) if case["sorted"] else torch.from_numpy(choices // case["top_k"]).to(device)
        x, w = state["x"][rows].double(), state["weight"][e].double()
        y[begin:end] = torch.mm(_exact_4_bits(x), _exact_4_bits(w).t())
        if train:
            g = state["grad"][begin:end].double()
            gx.index_add_(0, rows, torch.mm(_exact_4_bits(g), _exact_4_bits(w.t().contiguous()).t()))
            gw[e] = torch.mm(_exact_4_bits(g.t().contiguous()), _exact_4_bits(x.t().contiguous()).t())
    return (y, gx, gw) if train else y
