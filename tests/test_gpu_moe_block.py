"""The mixture-of-experts example: its gradients against plain autograd, and that it learns."""

from __future__ import annotations

import importlib.util
import os

import pytest
import torch

from adamw4bit_b200 import activations as A
from adamw4bit_b200 import routing as R

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_spec = importlib.util.spec_from_file_location("moe_block", os.path.join(ROOT, "examples", "moe_block.py"))
M = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(M)


def _plain(block, x, valid):
    """The block by torch's own operations in float64, choices as the router makes them."""
    with torch.no_grad():
        y = A.rms_norm(x, block.norm)
        e = R.route(torch.nn.functional.linear(y.float(), block.router), block.k, valid).experts.clamp(min=0).long()
    p = {n: t.detach().double().requires_grad_() for n, t in block.named_parameters()}
    x = x.double()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * p["norm"]

    def glu(z):
        g, u = z.chunk(2, -1)
        return torch.nn.functional.silu(g) * u

    out = glu(y @ p["shared_gate_up"].t()) @ p["shared_down"].t()
    prob = torch.softmax(y @ p["router"].t(), -1)
    w = prob.gather(1, e)
    w = w / w.sum(-1, keepdim=True)
    one = torch.nn.functional.one_hot(e, prob.shape[1]).double() * valid[:, None, None]
    for i in range(prob.shape[1]):
        out = out + (one[..., i] * w).sum(-1, keepdim=True) * (glu(y @ p["gate_up"][i].t()) @ p["down"][i].t())
    n = valid.sum()
    share = prob.shape[1] * one.sum((0, 1)) / (block.k * n)
    return x + out, (share * (prob * valid[:, None]).sum(0) / n).sum(), p


def test_gradients_match_plain_autograd():
    torch.manual_seed(3)
    block = M.MoEBlock(dim=192, hidden=160, experts=8, k=2)
    x = torch.randn(600, 192, device="cuda", dtype=torch.bfloat16)
    valid = torch.rand(600, device="cuda") >= 0.1
    c = torch.randn(600, 192, device="cuda", dtype=torch.bfloat16)
    got, balance = block(x, valid)
    ((got * c).sum() + 3.0 * balance).backward()
    want, want_balance, p = _plain(block, x, valid)
    ((want * c.double()).sum() + 3.0 * want_balance).backward()
    off = (got.double() - want).norm(dim=1) / want.norm(dim=1)
    assert (off > 0.02).sum() <= 12
    assert abs(balance.item() - want_balance.item()) <= 0.02 * want_balance.item()
    for name, t in block.named_parameters():
        a, b = t.grad.double(), p[name].grad
        # 8-bit checkpoints: a step is at most 1/64 of a block's largest value, rounding errors of
        # step / sqrt(12) average over the rows; bfloat16 products add 2^-8 each
        assert (a - b).norm() <= 0.06 * b.norm(), name


def test_learns():
    losses, balances = M.train(steps=40, tokens=2048, dim=256, hidden=256, experts=8)
    assert all(l == l and abs(l) < 1e6 for l in losses)
    assert losses[-1] < 0.75 * losses[0]
    assert max(balances[-5:]) < 1.5
