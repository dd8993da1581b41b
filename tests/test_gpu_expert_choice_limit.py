"""More choices per token than the way back can add up: refused before the work is done, where a gradient would need it."""

import pytest
import torch

from flex_shard_amd.experts import route_tokens
from flex_shard_amd.mxfp4 import mxfp4_expert_linear

pytestmark = pytest.mark.gpu


def test_more_than_64_choices(device):
    gen = torch.Generator(device=device).manual_seed(1)
    ids = torch.randint(0, 5, (3, 65), generator=gen, device=device)
    routing = route_tokens(ids, 5)
    x, w = torch.randn(3, 64, generator=gen, device=device), torch.randn(5, 40, 64, generator=gen, device=device)
    with pytest.raises(NotImplementedError, match="at most 64 choices"):
        mxfp4_expert_linear(x.clone().requires_grad_(), w, routing)
    # without a gradient for the tokens, and on sorted rows, any number will do
    y = mxfp4_expert_linear(x, w.requires_grad_(), routing)
    (gw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert torch.isfinite(gw).all()
    rows = x[routing.source.long() // 65].requires_grad_()
    again = mxfp4_expert_linear(rows, w, routing, sorted_rows=True)
    assert torch.equal(again, y)
    assert torch.autograd.grad(again, rows, torch.ones_like(y))[0].shape == rows.shape
    few = route_tokens(ids[:, :64].contiguous(), 5)
    leaf = x.clone().requires_grad_()
    assert torch.autograd.grad(mxfp4_expert_linear(leaf, w, few).sum(), leaf)[0].shape == x.shape
