"""Offsets of grouped_linear that do not lie within the rows: every pass takes the same rows for a group."""

from __future__ import annotations

import pytest
import torch

from adamw4bit_b200 import activations as A

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("offsets,bounds", [
    ([-5, 20, 45, 70], [0, 20, 45, 70]),
    ([-9, -5, 30, 70], [0, 0, 30, 70]),
    ([0, 20, 90, 200], [0, 20, 70, 70]),
    ([10, 20, 20, 50], [10, 20, 20, 50]),                 # rows of no group
], ids=str)
def test_offsets_are_cut_to_the_rows(offsets, bounds):
    g = torch.Generator().manual_seed(3)
    x = (torch.randint(-127, 128, (70, 64), generator=g) / 64).to(torch.bfloat16)
    x[:, ::32] = 1.5                                      # the checkpoint holds these values as they are
    w = torch.randn(3, 40, 64, generator=g).to(torch.bfloat16)
    c = torch.randn(70, 40, generator=g).to(torch.bfloat16)
    xs, ws = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    y = A.grouped_linear(xs, ws, torch.tensor(offsets, dtype=torch.int32, device=DEV))
    y.backward(c.to(DEV))
    want_y, want_x = torch.zeros(70, 40, dtype=torch.float64), torch.zeros(70, 64, dtype=torch.float64)
    want_w = torch.zeros(3, 40, 64, dtype=torch.float64)
    size_y, size_x, size_w = want_y.clone(), want_x.clone(), want_w.clone()
    xd, wd, cd = x.double(), w.double(), c.double()
    for i, (a, b) in enumerate(zip(bounds, bounds[1:])):
        want_y[a:b], size_y[a:b] = xd[a:b] @ wd[i].t(), xd[a:b].abs() @ wd[i].abs().t()
        want_x[a:b], size_x[a:b] = cd[a:b] @ wd[i], cd[a:b].abs() @ wd[i].abs()
        want_w[i], size_w[i] = cd[a:b].t() @ xd[a:b], cd[a:b].abs().t() @ xd[a:b].abs()
    for got, want, size in ((y, want_y, size_y), (xs.grad, want_x, size_x), (ws.grad, want_w, size_w)):
        # bfloat16's rounding, and a float32 sum of at most 70 terms that may be truncated at each
        assert ((got.detach().cpu().double() - want).abs() <= 1.02 * 2.0 ** -8 * want.abs() + 144 * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("offsets", [[0, 40, 20, 70], [0, 70, 0, 70], [60, 40, 20, 0]], ids=str)
def test_offsets_that_descend_are_refused(offsets):
    x = torch.ones(70, 64, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(3, 40, 64, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="ascend"):
        A.grouped_linear(x, w, torch.tensor(offsets, dtype=torch.int32, device=DEV))
