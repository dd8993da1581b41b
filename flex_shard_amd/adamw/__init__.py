"""AdamW for what Muon does not update (or for everything), many tensors at a time.

:class:`FlexShardAdamW` is a ``torch.optim.Optimizer`` whose step is one table of
tensors on the HIP kernels, with fp32 states or with 8-bit ones.  Clipping by the
gradients' norm is part of the step's one pass over them:

    square_sum = grad_square_sum([p.grad for p in params])   # all_reduce it over the ranks' shards
    optimizer.step(square_sum=square_sum, max_norm=1.0)
"""

from __future__ import annotations

from typing import Any, Iterable

import torch

from .. import _native, hip_ops
from .._native import ADAMW_BLOCK, DT_BF16, DT_F32

_DT = {torch.bfloat16: DT_BF16, torch.float32: DT_F32}


def grad_square_sum(grads: Iterable[torch.Tensor | None]) -> torch.Tensor:
    """The sum of the squares of the gradients' elements (bf16, fp16 or fp32, all on
    one GPU; None is left out), a float64 scalar there: the square of their
    common norm.  Products and sums in 64 bits, in an order that the sizes alone decide.  Of
    sharded gradients it is this rank's part: add the ranks' up before it is used."""
    present = [g if g.is_contiguous() else g.detach().contiguous() for g in grads if g is not None]
    if not present:
        raise ValueError("at least one gradient")
    return hip_ops.grad_square_sum(present)


class FlexShardAdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) on contiguous bf16 or fp32 parameters, each
    with a gradient of either type, all on one GPU.

    ``state_bits`` 32: ``exp_avg`` and ``exp_avg_sq`` are fp32 whatever the parameter's type.
    8: they are uint8 codes with fp32 scales for every 128 elements (``exp_avg_scale``,
    ``exp_avg_sq_scale``; :meth:`state_values` gives what they stand for): 2 1/16
    bytes an element for 8.  Arithmetic is in fp32, the parameter rounded once; with 8 bits the
    second moment's root and the moments' quotient are the hardware's, each to one unit in
    fp32's last place, and a second moment below 2**-126 may count as zero.  ``step`` is
    an int32 on the GPU, so that a captured step counts on; ``lr`` may be an fp32 scalar
    there, which a captured step reads anew.  A captured step keeps the addresses that it was
    captured with: load states, and take new gradients' memory, before.  Parameters without a gradient
    are left alone; parameters or states that overlap are refused, before anything is stepped."""

    def __init__(
        self, params, lr: float | torch.Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
        weight_decay: float = 1e-2, *, state_bits: int = 32,
    ) -> None:
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def add_param_group(self, param_group: dict[str, Any]) -> None:
        super().add_param_group(param_group)
        try:
            _check_group(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    # ------------------------------------------------------------------- states
    def _new_state(self, p: torch.Tensor, bits: int) -> dict[str, torch.Tensor]:
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            # the zeros would be part of the graph, and every replay would begin with them
            raise RuntimeError("the states of an AdamW step must exist before it is captured: run one step, or load them")
        blocks = -(-p.numel() // ADAMW_BLOCK)
        kind, device = torch.float32 if bits == 32 else torch.uint8, p.device
        state = {"step": torch.zeros((), dtype=torch.int32, device=device)}
        for name in ("exp_avg", "exp_avg_sq"):
            state[name] = torch.zeros(p.shape, dtype=kind, device=device)
            if bits == 8:
                state[f"{name}_scale"] = torch.zeros((blocks,), dtype=torch.float32, device=device)
        return state

    def state_values(self, param: torch.Tensor, dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
        """``exp_avg`` and ``exp_avg_sq`` of a parameter as numbers."""
        state = self.state.get(param)
        if not state:
            raise KeyError("this parameter has no state yet")
        if state["exp_avg"].dtype != torch.uint8:
            return state["exp_avg"].to(dtype, copy=True), state["exp_avg_sq"].to(dtype, copy=True)
        return hip_ops.adamw_state_values(
            state["exp_avg"], state["exp_avg_scale"], state["exp_avg_sq"], state["exp_avg_sq_scale"], dtype
        )

    def load_state_dict(self, state_dict: dict[str, Any]) -> None:
        """Copies of the saved states, of the types that they have here (``torch``'s
        own loading would cast them to the parameters').  Groups that name no ``state_bits``, ``torch``'s own
        AdamW's, have 32."""
        loaded: dict[torch.Tensor, dict[str, torch.Tensor]] = {}

        def take(_, state_dict: dict[str, Any]) -> dict[str, Any]:
            groups, states = [], dict(state_dict["state"])
            for group in state_dict["param_groups"]:
                group = {"state_bits": 32, **group}
                for option in ("amsgrad", "maximize"):
                    if group.get(option):
                        raise NotImplementedError(f"the AdamW kernels have no {option}")
                _check_group({**group, "params": ()})
                groups.append(group)
            if [len(g["params"]) for g in groups] == [len(g["params"]) for g in self.param_groups]:
                for group, saved in zip(self.param_groups, groups):
                    for p, index in zip(group["params"], saved["params"]):
                        if states.get(index):
                            state = states.pop(index)
                            loaded[p] = mine = self._copy_of(p, saved["state_bits"], state)
                            if len(state) > len(mine):  # (states of other names)
                                states[index] = {name: value for name, value in state.items() if name not in mine}
            return {**state_dict, "param_groups": groups, "state": states}

        def put(_) -> None:
            for p, state in loaded.items():
                self.state[p] = state | self.state.get(p, {})

        # (behind the hooks that change what is loaded, and ahead of those that look at it)
        handles = self.register_load_state_dict_pre_hook(take), self.register_load_state_dict_post_hook(put, prepend=True)
        try:
            super().load_state_dict(state_dict)
        finally:
            for handle in handles:
                handle.remove()

    def _copy_of(self, p: torch.Tensor, bits: int, saved: dict[str, Any]) -> dict[str, torch.Tensor]:
        state = self._new_state(p, bits)
        state["step"].fill_(int(saved["step"]))
        for name, mine in state.items():
            if name == "step":
                continue
            value = saved.get(name)
            if value is None or value.shape != mine.shape or (value.dtype == torch.uint8) != (mine.dtype == torch.uint8):
                got = None if value is None else f"{value.dtype} {tuple(value.shape)}"
                raise ValueError(f"{bits}-bit states need {name} as {mine.dtype} {tuple(mine.shape)}, got {got}")
            mine.copy_(value)
        return state

    # --------------------------------------------------------------------- step
    @torch.no_grad()
    def step(self, closure=None, *, square_sum: torch.Tensor | None = None, max_norm: float | None = None):
        """One step on the parameters' ``.grad``.  With ``square_sum`` (of
        :func:`grad_square_sum`) and ``max_norm`` the gradients are scaled by min(1, max_norm /
        (sqrt(square_sum) + 1e-6)) as they are read.  A ``square_sum`` that is an infinity
        or not a number leaves parameters, states and step counts as they are."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if max_norm is not None and (square_sum is None or not max_norm > 0):
            raise ValueError(f"clipping needs the gradients' square_sum and a positive max_norm, got {max_norm}")
        device, index = None, -1
        groups: list[tuple] = []
        table: list[int] = []
        stepped, copies = [], []  # (the queued kernels read the copies)
        states, strided, int32 = self.state, torch.strided, torch.int32
        for group in self.param_groups:
            lr, bits, number, begin = group["lr"], group["state_bits"], len(groups), len(table)
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if device is None:
                    device, index = p.device, p.get_device()
                    _check_sum(square_sum, device)
                param_dt, grad_dt = _DT.get(p.dtype), _DT.get(g.dtype)
                if (
                    param_dt is None or grad_dt is None or p.get_device() != index or g.get_device() != index or index < 0
                    or g.layout is not strided or g.shape != p.shape or not p.is_contiguous()
                ):
                    _refuse_pair(p, g, device)
                if not g.is_contiguous():
                    g = g.contiguous()
                    copies.append(g)
                state = states[p]
                if not state:
                    state.update(self._new_state(p, bits))
                m, v, count, numel = state["exp_avg"], state["exp_avg_sq"], state["step"], p.numel()
                # (they may have been replaced, or the parameter's memory since they were made)
                nbytes = numel if bits == 8 else 4 * numel
                if (
                    m.nbytes != nbytes or v.nbytes != nbytes or not m.is_contiguous() or not v.is_contiguous()
                    or m.get_device() != index or v.get_device() != index
                    or count.dtype is not int32 or count.nbytes != 4 or count.get_device() != index
                ):
                    _check_state(state, numel, bits, index)
                m_scale = v_scale = 0
                if bits == 8:
                    m_scale, v_scale = state["exp_avg_scale"], state["exp_avg_sq_scale"]
                    nbytes = 4 * -(-numel // ADAMW_BLOCK)
                    if (
                        m_scale.nbytes != nbytes or v_scale.nbytes != nbytes or not m_scale.is_contiguous() or not v_scale.is_contiguous()
                        or m_scale.get_device() != index or v_scale.get_device() != index
                    ):
                        _check_state(state, numel, bits, index)
                    m_scale, v_scale = m_scale.data_ptr(), v_scale.data_ptr()
                # (an fsh_adamw_tensor)
                table += (
                    p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), m_scale, v_scale, count.data_ptr(), numel,
                    param_dt, grad_dt, bits, number,
                )
                stepped.append(p)
            if len(table) == begin:  # (no gradients: nothing of the group is looked at)
                continue
            address = None
            if isinstance(lr, torch.Tensor):
                lr, address = _learning_rate(lr, device)
            groups.append((lr, address, *group["betas"], group["eps"], group["weight_decay"]))
        if stepped:
            hip_ops.adamw_step(table, groups, device, square_sum, max_norm or 0.0)  # (checks all of it before any of it is queued)
            torch.autograd.graph.increment_version(stepped)
        return loss


def _check_group(group: dict[str, Any]) -> None:
    beta1, beta2 = group["betas"]
    if not (0 <= beta1 < 1 and 0 <= beta2 < 1):
        raise ValueError(f"betas must be in [0, 1), got {group['betas']}")
    for name in ("eps", "weight_decay"):
        if not group[name] >= 0:
            raise ValueError(f"{name} must not be negative, got {group[name]}")
    if not isinstance(group["lr"], torch.Tensor) and not group["lr"] >= 0:
        raise ValueError(f"lr must not be negative, got {group['lr']}")
    if group["state_bits"] not in (8, 32):
        raise NotImplementedError(f"states have 8 or 32 bits, got {group['state_bits']}")
    for p in group["params"]:
        if p.dtype not in _DT:
            raise NotImplementedError(f"the AdamW kernels update bf16 or fp32 parameters, got {p.dtype}")


def _check_sum(square_sum: torch.Tensor | None, device: torch.device) -> None:
    if square_sum is not None and (square_sum.dtype != torch.float64 or square_sum.numel() != 1 or square_sum.device != device):
        raise ValueError(f"square_sum must be one float64 on {device}, got {square_sum.dtype} {tuple(square_sum.shape)} on {square_sum.device}")


def _refuse_pair(p: torch.Tensor, g: torch.Tensor, device: torch.device) -> None:
    """Why the kernels cannot take a parameter and its gradient."""
    if p.device.type != "cuda":
        raise RuntimeError("flex_shard_amd kernels run on the GPU only; there is no CPU path.")
    if p.dtype not in _DT or g.dtype not in _DT or g.layout != torch.strided:
        raise NotImplementedError(f"the AdamW kernels take dense bf16 or fp32 parameters and gradients, got {p.dtype} and {g.dtype} ({g.layout})")
    if p.device != device or g.device != device:
        raise ValueError(f"all parameters and gradients of a step must live on {device}, got {p.device} and {g.device}")
    raise ValueError(f"contiguous parameters with gradients of their shape, got {tuple(p.shape)} / {p.stride()} and {tuple(g.shape)}")


def _check_state(state: dict[str, torch.Tensor], numel: int, bits: int, index: int) -> None:
    """That a parameter's states are of its size and on its device, as the kernels take them."""
    kind = torch.float32 if bits == 32 else torch.uint8
    wanted = {"step": (torch.int32, 1), "exp_avg": (kind, numel), "exp_avg_sq": (kind, numel)}
    if bits == 8:
        wanted |= dict.fromkeys(("exp_avg_scale", "exp_avg_sq_scale"), (torch.float32, -(-numel // ADAMW_BLOCK)))
    for name, (dtype, count) in wanted.items():
        t = state[name]
        if t.dtype != dtype or t.numel() != count or not t.is_contiguous() or t.get_device() != index:
            raise ValueError(
                f"{bits}-bit states need {name} as {count} contiguous {dtype} where the parameter is, got {t.dtype} {tuple(t.shape)} on {t.device}"
            )


def _learning_rate(lr: torch.Tensor, device: torch.device) -> tuple[float, int | None]:
    """A learning rate in a tensor: as a number, and its address on the GPU."""
    if lr.numel() != 1:
        raise ValueError(f"lr must be one number, got {tuple(lr.shape)}")
    if lr.device.type == "cpu":
        return float(lr), None
    if lr.device != device or lr.dtype != torch.float32:
        raise ValueError(f"lr on the GPU must be fp32 on {device}, got {lr.dtype} on {lr.device}")
    return 0.0, lr.data_ptr()


__all__ = ["FlexShardAdamW", "grad_square_sum"]
