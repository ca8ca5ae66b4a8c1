"""The router over more rows than are resident, both directions, against float64 on the device.

Blocks stay and walk the rows with the next one on its way; here every group of lanes has two rows or more.
Sums of p: a lane adds at most 32 logits and 5 shuffles join them, so a probability is off by (37 + 6) 2^-24 and the
exponential's 1.25 * 2^-24 |l - max|; over rows a lane's own (under 16), 5 shuffles and 32 warps, then whole numbers of
2^-32 from block to block; the balance adds up to 4 products a thread, 5 shuffles and 32 warps.  That is 2^-24 * 160 and
the exponentials', under 2e-5: a single row of 40009 that were missing would be seen."""

from __future__ import annotations

import math

import pytest
import torch

from adamw4bit_b200 import routing as Q
from tests import act8_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
EPS32 = 2.0 ** -24
CASES = [(400003, 8, 2), (400003, 8, 8), (300007, 16, 4), (40009, 32, 8), (40009, 32, 32), (40009, 64, 8), (40009, 128, 10),
         (40009, 200, 12), (40009, 256, 32), (40009, 512, 3), (20011, 1000, 10), (20011, 1024, 32)]


@pytest.mark.parametrize("rows,experts,k", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_every_row_of_a_walk(renormalize, dtype, rows, experts, k):
    g = torch.Generator(DEV).manual_seed(rows + experts + k)
    logits = (1.5 * torch.randn(rows, experts, generator=g, device=DEV)).to(dtype)
    logits[11::101] = -math.inf
    valid = torch.ones(rows, dtype=torch.bool, device=DEV)
    valid[5::7] = False
    dw = torch.randn(rows, k, generator=g, device=DEV)
    r = Q.route_forward(logits, k, valid=valid, renormalize=renormalize)
    dl = Q.route_backward(dw, torch.full((), 0.5, device=DEV), r)

    live = valid.clone()
    live[11::101] = False
    l = torch.where(live[:, None], logits.double(), 0.0)
    at = l.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    chosen = torch.where(live[:, None], at, -1)
    assert torch.equal(r.experts.long(), chosen)
    counts = torch.bincount(at[live].flatten(), minlength=experts)
    assert torch.equal(r.counts.long(), counts)
    p = torch.softmax(l, -1) * live[:, None]
    span = (l.amax(-1, keepdim=True) - l).amax().item()
    one = (43 + 1.25 * span + 4) * EPS32                              # relative error of a probability
    total = p.gather(1, at).sum(-1, keepdim=True).clamp(min=1e-300) if renormalize else torch.ones_like(p[:, :1])
    w = p.gather(1, at) / total
    assert ((r.weights.double() - w).abs() <= 2 * one * w).all()
    n = live.sum().double()
    share = experts * counts.double() / (k * n)
    balance = (share * p.sum(0) / n).sum().item()
    lean = ((l.amax(-1, keepdim=True) - l) * p).sum(-1).amax().item()     # of the exponentials, weighted as the sum weights them
    assert abs(r.balance_loss.item() - balance) <= (160 + 2.5 * lean) * EPS32 * balance

    d = dw.double() * live[:, None]
    inner = (w * d).sum(-1, keepdim=True)
    t = w * (d - inner) if renormalize else w * d
    u = share * 0.5 / n
    back = (p * u).sum(-1, keepdim=True) + (0.0 if renormalize else inner)
    want = (p * (u - back)).scatter_add(1, at, t)
    size = p * (u + (p * u).sum(-1, keepdim=True))
    wd = (w * d).abs()
    if not renormalize:
        size = size + p * wd.sum(-1, keepdim=True)
    size = size.scatter_add(1, at, wd + w * wd.sum(-1, keepdim=True))
    slack = (4 * one + (k + 43) * EPS32) * size + 1e-37
    off = (dl.double() - want).abs() - (1.02 * R.UNIT[dtype] * want.abs() + R.STEP[dtype] + slack)
    assert off.max() <= 0
    assert not dl[~live].any()
