"""A mixture-of-experts layer in microscaled 4-bit products: trained, then served.

    PYTHONPATH=. python examples/mxfp4_experts.py [--tokens T] [--dim D] [--hidden H] [--experts E] [--top-k K] [--steps N]

The layer is a router, gated experts and one shared expert that every token takes.
Training keeps bf16 parameters and quantizes within the call; serving quantizes
them once and multiplies the tokens' rows without sorting copies of them.
"""

from __future__ import annotations

import argparse

import torch
from torch import nn
from torch.nn import functional as F

from flex_shard_amd.experts import combine_tokens, dispatch_tokens, route_tokens
from flex_shard_amd.mxfp4 import FlexShardMxFp4Linear, mxfp4_expert_linear, mxfp4_linear, quantize_mxfp4_weight


class ExpertLayer(nn.Module):
    def __init__(self, dim: int, hidden: int, experts: int, top_k: int, device: str = "cuda", dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        self.experts, self.top_k = experts, top_k
        made = dict(device=device, dtype=dtype)
        self.router = nn.Linear(dim, experts, bias=False, device=device)
        self.gate = nn.Parameter(torch.randn(experts, hidden, dim, **made) * dim**-0.5)
        self.up = nn.Parameter(torch.randn(experts, hidden, dim, **made) * dim**-0.5)
        self.down = nn.Parameter(torch.randn(experts, dim, hidden, **made) * hidden**-0.5)
        self.shared_up = FlexShardMxFp4Linear(dim, hidden, bias=True, **made)
        self.shared_down = FlexShardMxFp4Linear(hidden, dim, bias=True, **made)

    def choose(self, x: torch.Tensor):
        weights, ids = torch.softmax(self.router(x.float()), dim=-1).topk(self.top_k, dim=-1)
        return route_tokens(ids, self.experts), weights / weights.sum(dim=-1, keepdim=True)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        routing, weights = self.choose(x)
        # sorted once for both projections: one sum over a token's choices brings both gradients back
        rows = dispatch_tokens(x, routing)
        gate = mxfp4_expert_linear(rows, self.gate, routing, sorted_rows=True)
        up = mxfp4_expert_linear(rows, self.up, routing, sorted_rows=True)
        down = mxfp4_expert_linear(F.silu(gate) * up, self.down, routing, sorted_rows=True)
        return combine_tokens(down, routing, weights) + self.shared_down(F.silu(self.shared_up(x)))

    def quantized(self) -> "ServedExperts":
        return ServedExperts(self)


class ServedExperts:
    """The layer with its weights quantized once."""

    def __init__(self, layer: ExpertLayer) -> None:
        self.layer = layer
        self.gate, self.up, self.down = (quantize_mxfp4_weight(w.detach()) for w in (layer.gate, layer.up, layer.down))
        self.shared_up, self.shared_down = (quantize_mxfp4_weight(m.weight.detach()) for m in (layer.shared_up, layer.shared_down))

    @torch.no_grad()
    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        routing, weights = self.layer.choose(x)
        gate = mxfp4_expert_linear(x, self.gate, routing)
        up = mxfp4_expert_linear(x, self.up, routing)
        down = mxfp4_expert_linear(F.silu(gate) * up, self.down, routing, sorted_rows=True)
        shared = mxfp4_linear(F.silu(mxfp4_linear(x, self.shared_up, self.layer.shared_up.bias)), self.shared_down, self.layer.shared_down.bias)
        return combine_tokens(down, routing, weights) + shared


def train(layer: ExpertLayer, x: torch.Tensor, target: torch.Tensor, steps: int, lr: float = 2e-3) -> list[float]:
    """Mean squared errors before each of the steps, and after the last."""
    optimizer = torch.optim.Adam(layer.parameters(), lr=lr)
    losses = []
    for step in range(steps + 1):
        loss = F.mse_loss(layer(x).float(), target)
        losses.append(loss.item())
        if step < steps:
            optimizer.zero_grad()
            loss.backward()
            optimizer.step()
    return losses


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("tokens", 512), ("dim", 512), ("hidden", 1024), ("experts", 8), ("top-k", 2), ("steps", 20)):
        parser.add_argument(f"--{name}", type=int, default=value)
    args = parser.parse_args()
    torch.manual_seed(0)
    layer = ExpertLayer(args.dim, args.hidden, args.experts, args.top_k)
    x = torch.randn(args.tokens, args.dim, device="cuda", dtype=torch.bfloat16)
    losses = train(layer, x, torch.tanh(x.float().roll(1, dims=-1)), args.steps)
    print(f"error before training {losses[0]:.4f}, after {args.steps} steps {losses[-1]:.4f}")
    served = layer.quantized()
    for tokens in (1, 16, args.tokens):
        with torch.no_grad():
            want = layer(x[:tokens]).float()
        got = served(x[:tokens]).float()
        print(f"{tokens} tokens served: largest difference {(got - want).abs().max().item():.2e} of {want.abs().max().item():.2e}")


if __name__ == "__main__":
    main()
