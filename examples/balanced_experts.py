"""A layer of routed experts whose loads are kept even by entropic transport, trained with a Sinkhorn divergence.

    python examples/balanced_experts.py [--steps N] [--tokens T] [--experts E] [--norm] [--orthogonal]

Points of a mixture are moved onto another cloud by ``y = x + experts(x)``. In every step the alternating solver gives one
price per expert (:func:`flash_sinkhorn_b200.experts.transport_bias`) at which a transport plan from the tokens to the
router's rows fills all experts alike; the router's choice takes logits plus prices, the gates the logits alone. The
layer is :func:`flash_sinkhorn_b200.experts.expert_mlp`, which keeps its inner activations in 8 bits for the backward
pass, and the loss is the debiased divergence between ``y`` and the target cloud. ``--norm`` puts
:func:`flash_sinkhorn_b200.experts.layer_norm` in front of the experts, and ``--orthogonal`` updates their matrices by
:func:`flash_sinkhorn_b200.experts.orthogonalize` of the gradients' momentum instead of Adam.
"""
import argparse
import os
import sys

import torch

if __name__ == "__main__":
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from flash_sinkhorn_b200 import SamplesLoss
from flash_sinkhorn_b200.experts import Routing, expert_mlp, layer_norm, orthogonalize, route_tokens, transport_bias


class BalancedExperts(torch.nn.Module):
    """``x + experts(x)`` with ``slots`` of ``experts`` gated experts per token, ``x + experts(norm(x))`` with ``norm``. Master
    weights are fp32, products bf16."""

    def __init__(self, width: int, inner: int, experts: int, slots: int, eps: float = 0.5, balance: bool = True, norm: bool = False):
        super().__init__()
        self.scale = torch.nn.Parameter(torch.ones(width)) if norm else None
        self.shift = torch.nn.Parameter(torch.zeros(width)) if norm else None
        self.slots, self.eps, self.balance = slots, eps, balance
        self.router = torch.nn.Parameter(torch.randn(experts, width) * width**-0.5)
        self.w_in = torch.nn.Parameter(torch.randn(experts, 2 * inner, width) * width**-0.5)
        self.w_out = torch.nn.Parameter(torch.randn(experts, width, inner) * 0.1 * inner**-0.5)

    def route(self, x: torch.Tensor) -> Routing:
        logits = x.float() @ self.router.t()
        prices = transport_bias(x, self.router, eps=self.eps, n_iters=50) if self.balance else None
        return route_tokens(logits, self.slots, bias=prices)

    def forward(self, x: torch.Tensor):
        routing = self.route(x)
        h = x.bfloat16() if self.scale is None else layer_norm(x.bfloat16(), self.scale, self.shift)
        y = expert_mlp(h, self.w_in.bfloat16(), self.w_out.bfloat16(), routing)
        return x + y.float(), routing


class OrthogonalUpdates(torch.optim.Optimizer):
    """Matrices ``[.., N, K]`` moved against their gradients' momentum with all singular values brought to about 1."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.9):
        super().__init__(params, dict(lr=lr, momentum=momentum))

    @torch.no_grad()
    def step(self):
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                m = self.state[p].setdefault("momentum", torch.zeros_like(p))
                m.mul_(group["momentum"]).add_(p.grad)
                n, k = p.shape[-2:]
                p.add_(orthogonalize(m).float(), alpha=-group["lr"] * max(1.0, n / k) ** 0.5)


def clouds(tokens: int, width: int, seed: int = 0):
    """A mixture of four Gaussians with uneven weights, and the cloud that each of them is to be moved to."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    centres = 2.0 * torch.randn(4, width, generator=gen, device="cuda")
    targets = centres.roll(1, 0) * 0.5
    part = torch.multinomial(torch.tensor([0.55, 0.25, 0.15, 0.05], device="cuda"), tokens, True, generator=gen)
    noise = lambda: 0.3 * torch.randn(tokens, width, generator=gen, device="cuda")
    return centres[part] + noise(), targets[part] + noise()


def train(steps: int = 60, tokens: int = 2048, width: int = 64, inner: int = 128, experts: int = 8, slots: int = 2,
          balance: bool = True, verbose: bool = False, norm: bool = False, orthogonal: bool = False):
    """Losses of all steps, and the share of the pairs that the busiest expert has in the last one, times the experts."""
    torch.manual_seed(0)
    layer = BalancedExperts(width, inner, experts, slots, balance=balance, norm=norm).cuda()
    x, target = clouds(tokens, width)
    divergence = SamplesLoss("sinkhorn", blur=1.0, use_epsilon_scaling=False, eps=1.0, n_iters=30, half_cost=True)
    matrices = [layer.w_in, layer.w_out] if orthogonal else []
    rest = [p for p in layer.parameters() if not any(p is m for m in matrices)]
    optimisers = [torch.optim.Adam(rest, lr=1e-2)] + ([OrthogonalUpdates(matrices)] if orthogonal else [])
    losses = []
    for step in range(steps):
        y, routing = layer(x)
        loss = divergence(y, target)
        for optimiser in optimisers:
            optimiser.zero_grad()
        loss.backward()
        for optimiser in optimisers:
            optimiser.step()
        losses.append(loss.detach())
        if verbose and step % 10 == 0:
            load = routing.offsets.diff().float()
            print(f"step {step:3d}  divergence {loss.item():8.4f}  loads {load.min().item():.0f} to {load.max().item():.0f} "
                  f"of {tokens * slots / experts:.0f}")
    with torch.no_grad():
        load = layer.route(x).offsets.diff().float()
    return torch.stack(losses).tolist(), (load.max() / load.sum() * experts).item()


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--tokens", type=int, default=2048)
    parser.add_argument("--experts", type=int, default=8)
    parser.add_argument("--unbalanced", action="store_true", help="route by the logits alone")
    parser.add_argument("--norm", action="store_true", help="layer norm in front of the experts")
    parser.add_argument("--orthogonal", action="store_true", help="orthogonal updates of the experts' matrices")
    args = parser.parse_args()
    history, busiest = train(args.steps, args.tokens, experts=args.experts, balance=not args.unbalanced, verbose=True, norm=args.norm,
                             orthogonal=args.orthogonal)
    print(f"divergence {history[0]:.4f} -> {history[-1]:.4f}, busiest expert {busiest:.2f} times its share")
