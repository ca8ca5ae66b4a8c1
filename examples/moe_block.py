"""A mixture-of-experts block trained with 4-bit moments and 8-bit activation checkpoints.

    python examples/moe_block.py [--steps 30] [--tokens 4096]

The block is a norm, a router, E gated feed-forward experts of which every token visits k, and a
shared feed-forward that every token visits.  What waits for the backward pass is held in 8 bits: the
norm's input, gate and up of every feed-forward, and the inputs of all projections (the norm and the
gated activation write the checkpoints that the projections behind them keep).  The router's counts
are the groups of the experts' weight gradients, its balance loss keeps them even, and
``ZEEDENAdamW4Bit`` takes the step.  The task is synthetic: to reproduce a fixed random block.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

from adamw4bit_b200 import ZEEDENAdamW4Bit  # noqa: E402
from adamw4bit_b200 import activations as A  # noqa: E402
from adamw4bit_b200 import routing as R  # noqa: E402


def by_expert(experts: torch.Tensor, counts: torch.Tensor):
    """Choices in the experts' order: (choice of each row, offsets of the experts' rows)."""
    offsets = R.group_offsets(counts)
    flat = experts.flatten()
    order = torch.where(flat < 0, counts.numel(), flat).argsort(stable=True)     # no choice: behind all
    return order[: int(offsets[-1])], offsets


class MoEBlock(nn.Module):
    def __init__(self, dim=512, hidden=1024, experts=8, k=2, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.k = k

        def weight(*shape):
            return nn.Parameter(torch.randn(*shape, device=device, dtype=torch.float32).mul_(shape[-1] ** -0.5).to(dtype))

        self.norm = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))
        self.router = nn.Parameter(torch.randn(experts, dim, device=device) * dim ** -0.5)
        self.gate_up = weight(experts, 2 * hidden, dim)
        self.down = weight(experts, dim, hidden)
        self.shared_gate_up = weight(2 * hidden, dim)
        self.shared_down = weight(dim, hidden)

    def forward(self, x: torch.Tensor, valid: torch.Tensor | None = None):
        """x [tokens, dim] -> (x + the block's output, balance loss)"""
        y, y8 = A.rms_norm(x, self.norm, checkpoint_output=True)
        h, h8 = A.swiglu(A.linear(y, self.shared_gate_up, x8=y8), checkpoint_output=True)
        out = A.linear(h, self.shared_down, x8=h8)
        routed = R.route(nn.functional.linear(y.float(), self.router), self.k, valid=valid)
        choice, offsets = by_expert(routed.experts, routed.counts)
        token = choice // self.k
        h, h8 = A.swiglu(A.grouped_linear(y[token], self.gate_up, offsets), checkpoint_output=True)
        parts = A.grouped_linear(h, self.down, offsets, x8=h8)
        parts = parts * routed.weights.flatten()[choice, None].to(parts.dtype)
        return x + out + torch.zeros_like(out).index_add(0, token, parts), routed.balance_loss


def train(steps: int = 30, tokens: int = 4096, dim: int = 512, hidden: int = 1024, experts: int = 8, seed: int = 0,
          balance_weight: float = 0.01):
    """Losses of the steps, and the balance losses."""
    torch.manual_seed(seed)
    target, block = MoEBlock(dim, hidden, experts), MoEBlock(dim, hidden, experts)
    optimizer = ZEEDENAdamW4Bit(block.parameters(), lr=2e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.0)
    valid = torch.rand(tokens, device="cuda") >= 0.05
    losses, balances = [], []
    for _ in range(steps):
        x = torch.randn(tokens, dim, device="cuda", dtype=torch.bfloat16)
        with torch.no_grad():
            want, _ = target(x, valid)
        got, balance = block(x, valid)
        loss = (got.float() - want.float()).square().mean()
        (loss + balance_weight * balance).backward()
        optimizer.step()
        optimizer.zero_grad(set_to_none=True)
        losses.append(loss.detach())
        balances.append(balance.detach())
    return torch.stack(losses).tolist(), torch.stack(balances).tolist()


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--tokens", type=int, default=4096)
    a = ap.parse_args()
    losses, balances = train(a.steps, a.tokens)
    for i in range(0, a.steps, max(1, a.steps // 10)):
        print(f"step {i:4d}  loss {losses[i]:.4f}  balance {balances[i]:.3f}")
    print(f"last       loss {losses[-1]:.4f}  balance {balances[-1]:.3f}")
