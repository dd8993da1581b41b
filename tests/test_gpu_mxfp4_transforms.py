"""Function transforms and forward-mode derivatives of the 4-bit and expert layers are not implemented, and a call that
would need one is refused, with gradients on or off."""

import pytest
import torch
from torch.autograd import forward_ad

from flex_shard_amd.experts import combine_tokens, dispatch_tokens, route_tokens
from flex_shard_amd.mxfp4 import mxfp4_expert_linear, mxfp4_linear, quantize_mxfp4_weight

pytestmark = pytest.mark.gpu


def _calls(device):
    gen = torch.Generator(device=device).manual_seed(1)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=device)

    routing = route_tokens(torch.randint(0, 3, (6, 2), generator=gen, device=device), 3)
    w, stack, frozen = normal(40, 64), normal(3, 40, 64), quantize_mxfp4_weight(normal(40, 64), transposed=True)
    return {  # a call of one tensor, and the tensor
        "linear x": (lambda t: mxfp4_linear(t, w), normal(6, 64)),
        "linear weight": (lambda t: mxfp4_linear(w[:6], t), normal(40, 64)),
        "linear bias": (lambda t: mxfp4_linear(w[:6], w, t), normal(40)),
        "frozen x": (lambda t: mxfp4_linear(t, frozen), normal(6, 64)),
        "experts x": (lambda t: mxfp4_expert_linear(t, stack, routing), normal(6, 64)),
        "experts weight": (lambda t: mxfp4_expert_linear(w[:6], t, routing), normal(3, 40, 64)),
        "dispatch": (lambda t: dispatch_tokens(t, routing), normal(6, 64)),
        "combine rows": (lambda t: combine_tokens(t, routing, w[:6, :2]), normal(12, 64)),
        "combine weights": (lambda t: combine_tokens(w[:12], routing, t), normal(6, 2)),
    }


NAMES = ["linear x", "linear weight", "linear bias", "frozen x", "experts x", "experts weight", "dispatch", "combine rows", "combine weights"]


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_a_dual_tensor_is_refused(device, name, grad_mode):
    call, t = _calls(device)[name]
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        plain = call(t)  # plain tensors in a dual level are not
        with pytest.raises(NotImplementedError):
            call(forward_ad.make_dual(t, torch.ones_like(t)))
    assert torch.equal(plain, call(t))


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_function_transforms_are_refused(device, name, grad_mode):
    call, t = _calls(device)[name]
    with torch.set_grad_enabled(grad_mode):
        for transformed in (torch.vmap(call), torch.func.grad(lambda u: call(u[0]).sum()), lambda u: torch.func.jvp(lambda v: call(v[0]), (u,), (u,))):
            with pytest.raises(RuntimeError):
                transformed(t[None])
