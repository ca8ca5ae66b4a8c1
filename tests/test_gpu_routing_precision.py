"""Weights and float32 gradients of logits that are far apart.

Logits are whole steps below a top of zero, so that l - top is exact, and what remains is the exponential's own error:
2^-23 (one unit in the last place) where it is a full float32, else 2^-22 and 1.25 * 2^-24 |l - top|.  A total of n terms adds
n 2^-24 of itself; a division and a product 2^-24 each."""

from __future__ import annotations

import pytest
import torch

from adamw4bit_b200 import routing as Q

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
EPS32 = 2.0 ** -24
CASES = [(8, 8), (16, 12), (60, 32), (128, 8), (300, 20)]


def _far_apart(rows, experts, dtype):
    g = torch.Generator().manual_seed(experts)
    l = -(torch.rand(rows, experts, generator=g) * 80 * 4096).round() / 4096
    l[torch.arange(rows), torch.randint(experts, (rows,), generator=g)] = 0.0
    return l.to(dtype).to(DEV)


@pytest.mark.parametrize("experts,k", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_weights(renormalize, dtype, experts, k):
    l = _far_apart(700, experts, dtype)
    r = Q.route_forward(l, k, renormalize=renormalize)
    p = torch.softmax(l.double(), -1)
    w = p.gather(1, r.experts.long())
    slack = 2.0 + 2.0 + experts + 2.0 + 2.0
    if renormalize:
        w = w / w.sum(-1, keepdim=True)
    elif dtype != torch.float32:
        slack = slack + 2.0 + 1.25 * (p * l.double().abs()).sum(-1, keepdim=True)
    assert ((r.weights.double() - w).abs() <= slack * EPS32 * w).all()


@pytest.mark.parametrize("experts", [8, 16, 60, 300])
def test_float32_gradient(experts):
    l = _far_apart(700, experts, torch.float32)
    r = Q.route_forward(l, 1, renormalize=False)
    dl = Q.route_backward(torch.ones(700, 1, device=DEV), None, r).double()
    p = torch.softmax(l.double(), -1)
    top = r.experts.long()
    # d w / d l_e = -p_e w beside the choice: two probabilities and their product
    want = -p * p.gather(1, top)
    off = ((dl - want).abs() / want.abs()).scatter(1, top, 0.0)
    assert off.max() <= (2 * (experts + 6) + 4) * EPS32
