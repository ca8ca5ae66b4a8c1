"""A large weight gradient, over and over: the same bits each time, and right.

What a pair of blocks hands over late would show in single tiles of single runs only, so every run is
compared as a whole, with other inputs' runs between that leave other values in the blocks' memory."""

from __future__ import annotations

import pytest
import torch

from adamw4bit_b200 import activations as A

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
EPS32 = 2.0 ** -24


@pytest.mark.parametrize("rows,n,k,counts,dtype", [
    (8192, 14336, 4096, None, torch.bfloat16),                                   # cut tiles, several rounds
    (4096, 4096, 4096, None, torch.float16),                                     # whole tiles
    (8192, 2816, 1024, [700, 0, 1300, 64, 2000, 3, 1821, 2304], torch.float16),  # groups
], ids=str)
def test_every_run_has_the_same_bits(rows, n, k, counts, dtype):
    g = torch.Generator(DEV).manual_seed(rows + n)
    offsets = None
    if counts:
        offsets = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    inputs = []
    for _ in range(2):
        x = torch.randn(rows, k, generator=g, device=DEV).to(dtype)
        dy = (0.1 * torch.randn(rows, n, generator=g, device=DEV)).to(dtype)
        inputs.append((dy, A.quantize_act8(x)))
    first = [A.weight_grad(dy, x8, offsets).view(torch.int16) for dy, x8 in inputs]
    differ = torch.zeros((), dtype=torch.int64, device=DEV)
    for i in range(60):
        dy, x8 = inputs[i % 2]
        differ += (A.weight_grad(dy, x8, offsets).view(torch.int16) != first[i % 2]).sum()
    assert differ.item() == 0
    # some of its rows from the definition in float64: half a unit of the dtype, and a sum of `rows` terms that a
    # tensor core may truncate at each of them
    unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    at = torch.randperm(n, generator=g, device=DEV)[:48]
    (dy, x8), got = inputs[0], first[0].view(dtype)
    v, d = x8.dequantize().double(), dy[:, at].double()
    bounds = [0, rows] if offsets is None else offsets.tolist()
    for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
        ref, mag = d[a:b].t() @ v[a:b], d[a:b].abs().t() @ v[a:b].abs()
        mine = (got if offsets is None else got[e])[at].double()
        assert ((mine - ref).abs() <= 1.02 * unit * ref.abs() + 2.0 ** -24 + 2 * (b - a + 2) * EPS32 * mag).all()
