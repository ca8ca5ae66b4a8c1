"""The expert router and its gradients, against 64-bit definitions.

Indices and counts are exact.  Weights, the loss and gradients are float32 evaluations: exp and its
argument round by (4 + |l - max|) 2^-23 of the value, sums of n terms by n 2^-24 of their magnitudes,
and a gradient of the logits' dtype by half a unit in its last place.
"""

from __future__ import annotations

import math

import pytest
import torch

from adamw4bit_b200 import routing as Q
from tests import act8_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS32 = 2.0 ** -24


def _ids(v):
    return str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None


def _logits(rows, experts, dtype, seed=0, scale=1.5):
    g = torch.Generator().manual_seed(seed + rows * 1024 + experts)
    return (torch.randn(rows, experts, generator=g) * scale).to(dtype)


def _check(logits, k, valid, renormalize, dweights=None, dbalance=0.5, device_logits=None):
    rows, experts = logits.shape
    on = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    r = Q.route_forward(on(logits) if device_logits is None else device_logits, k, valid=on(valid),
                        renormalize=renormalize)
    db = torch.tensor(dbalance, device=DEV)
    dl = Q.route_backward(on(dweights), db, r).cpu()
    weights, chosen, counts, balance, ref = R.route(logits, k, valid, renormalize, dweights, dbalance)
    assert r.experts.dtype == r.counts.dtype == torch.int32 and dl.dtype == logits.dtype
    assert torch.equal(r.experts.cpu().long(), chosen)
    assert torch.equal(r.counts.cpu().long(), counts)
    span = 4 + (logits.double().nan_to_num(0, 0, 0).abs().amax().item() * 2)
    one = (2 * span + experts) * EPS32                       # relative error of a probability
    got = r.weights.cpu().double()
    bad = torch.isnan(weights)
    assert torch.equal(torch.isnan(got), bad)
    assert ((got - weights).abs() <= (2 * one * weights.abs() + 1e-37))[~bad].all()
    if torch.isnan(balance):
        assert torch.isnan(r.balance_loss).item()
    else:
        assert abs(r.balance_loss.item() - balance.item()) <= (one + (rows + experts + 8) * EPS32) * balance.item()
    live = chosen[:, 0] >= 0
    n = max(1, int(live.sum()))
    # every term of a gradient is p or w times something of these sizes
    p = torch.softmax(torch.where(live[:, None], logits.double(), 0.0), -1)
    share = experts * counts.double() / (k * n) * abs(dbalance) / n
    size = p * (share + (p * share).sum(-1, keepdim=True))
    if dweights is not None:
        wd = (weights * dweights.double()).abs()
        size += (p * wd.sum(-1, keepdim=True)) if not renormalize else 0.0
        picked = torch.zeros_like(p).scatter_add(1, chosen.clamp(min=0), wd + weights * wd.sum(-1, keepdim=True))
        size += picked
    slack = (4 * one + (k + experts) * EPS32) * size + 1e-37
    bad = torch.isnan(ref)
    assert torch.equal(torch.isnan(dl.double()), bad)
    off = (dl.double() - ref).abs() - (1.02 * R.UNIT[logits.dtype] * ref.abs() + R.STEP[logits.dtype] + slack)
    assert off[~bad].numel() == 0 or off[~bad].max() <= 0
    return r, dl


CASES = [(1, 1, 1), (1, 4, 2), (3, 8, 2), (50, 8, 8), (33, 13, 3), (70, 16, 4), (65, 31, 5), (40, 33, 32), (129, 64, 8),
         (37, 100, 7), (60, 128, 8), (20, 160, 6), (31, 256, 8), (9, 257, 4), (7, 512, 22), (5, 1000, 10), (4, 1024, 32)]


@pytest.mark.parametrize("rows,experts,k", CASES)
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_route(dtype, rows, experts, k):
    logits = _logits(rows, experts, dtype)
    g = torch.Generator().manual_seed(rows)
    dw = torch.randn(rows, k, generator=g)
    for renormalize in (True, False):
        _check(logits, k, None, renormalize, dw)
        _check(logits, k, torch.rand(rows, generator=g) < 0.7, renormalize, dw)
    _check(logits, k, None, True, None)


@pytest.mark.parametrize("experts", [8, 24, 128, 300])
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_ties_go_to_the_lowest_index(dtype, experts):
    logits = _logits(40, experts, dtype)
    logits[0] = 0.0
    logits[1] = torch.finfo(dtype).min
    logits[2] = torch.finfo(dtype).max
    logits[3, ::2], logits[3, 1::2] = 0.0, -0.0           # equal numbers
    logits[4:20] = (logits[4:20] * 2).round() / 2
    r, _ = _check(logits, 4, None, True, torch.ones(40, 4))
    assert r.experts[:4].tolist() == [[0, 1, 2, 3]] * 4


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_masked_experts_and_empty_rows(dtype):
    logits = _logits(30, 40, dtype)
    logits[:, 11:] = -math.inf
    logits[3, 2:] = -math.inf                             # fewer experts than choices
    logits[4] = -math.inf                                 # none
    logits[5, 1:] = -math.inf
    dw = torch.randn(30, 4, generator=torch.Generator().manual_seed(1))
    valid = torch.ones(30, dtype=torch.bool)
    valid[7] = False
    for renormalize in (True, False):
        r, dl = _check(logits, 4, valid, renormalize, dw)
        assert r.experts[3].tolist()[2:] == [-1, -1] and r.experts[4].tolist() == [-1] * 4
        assert not dl[4].any() and not dl[7].any() and not r.weights[4].any()


def test_nothing_valid():
    logits = _logits(9, 16, torch.float32)
    r, dl = _check(logits, 2, torch.zeros(9, dtype=torch.bool), True, torch.ones(9, 2))
    assert r.balance_loss.item() == 0.0 and not r.counts.any() and not dl.any()
    r = Q.route_forward(torch.empty(0, 16, device=DEV), 2)
    assert r.balance_loss.item() == 0.0 and not r.counts.any() and r.weights.shape == (0, 2)
    assert Q.route_backward(None, None, r).shape == (0, 16)


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_bad_values_behind_the_mask_do_not_leak(dtype):
    logits = _logits(20, 24, dtype)
    logits[3], logits[8, 5], logits[9, 2] = math.nan, math.inf, math.nan
    valid = torch.ones(20, dtype=torch.bool)
    valid[[3, 8, 9]] = False
    r, dl = _check(logits, 3, valid, False, torch.ones(20, 3))
    assert torch.isfinite(r.balance_loss).item() and torch.isfinite(dl).all()
    valid[9] = True                                       # a NaN that counts is seen
    r = Q.route_forward(logits.to(DEV), 3, valid=valid.to(DEV))
    assert r.experts[9, 0].item() == 2 and torch.isnan(r.weights[9]).all() and torch.isnan(r.balance_loss).item()
    assert torch.isfinite(r.weights[:9]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_strides(dtype):
    wide = _logits(60, 90, dtype).to(DEV)
    for view in (wide[:, 8:72], wide[::2, 3:60], wide.t(), wide[:1, :40].expand(7, 40)):
        dense = view.cpu().contiguous()
        _check(dense, 3, None, True, torch.ones(dense.shape[0], 3), device_logits=view)
    r = Q.route(wide.view(3, 20, 90), 5, valid=torch.ones(3, 20, dtype=torch.bool, device=DEV))
    assert r.weights.shape == r.experts.shape == (3, 20, 5)


def test_many_rows_are_reproducible():
    logits = _logits(30000, 64, torch.bfloat16).to(DEV)
    first, second = (Q.route_forward(logits, 6, renormalize=False) for _ in range(2))
    assert first.balance_loss.item() == second.balance_loss.item()
    assert first.counts.sum().item() == 30000 * 6
    p = torch.softmax(logits.double(), -1)
    top = torch.sort(logits.double(), dim=-1, descending=True, stable=True).indices[:, :6]
    assert torch.equal(first.experts.long(), top)
    share = 64 * first.counts.double() / (6 * 30000)
    want = (share * p.mean(0)).sum().item()
    assert abs(first.balance_loss.item() - want) <= 600 * EPS32 * want


@pytest.mark.parametrize("renormalize", [True, False])
def test_gradient_against_differences(renormalize):
    logits = _logits(12, 10, torch.float32, seed=5)
    c, d = torch.randn(12, 3, generator=torch.Generator().manual_seed(2)).double(), _logits(12, 10, torch.float32, seed=9)
    x = logits.to(DEV).requires_grad_()
    out = Q.route(x, 3, renormalize=renormalize)
    ((out.weights * c.float().to(DEV)).sum() + 2.5 * out.balance_loss).backward()

    def f(l):
        w, _, _, balance, _ = R.route(l, 3, None, renormalize)
        return ((w * c).sum() + 2.5 * balance).item()

    h = 1e-6                       # the choices stay as they are: logits are further apart than this
    top = torch.sort(logits, -1, descending=True).values
    assert (top[:, :3] - top[:, 1:4]).min() > 1e-4
    want = (f(logits.double() + h * d.double()) - f(logits.double() - h * d.double())) / (2 * h)
    terms = x.grad.cpu().double() * d.double()
    # h^2 times a third derivative of order 100, cancellation 1e-15 / h, the gradient float32
    assert abs(terms.sum().item() - want) <= 1e-8 + 100 * EPS32 * terms.abs().sum().item()


def test_unused_outputs_have_no_gradient():
    x = _logits(6, 8, torch.float32).to(DEV).requires_grad_()
    Q.route(x, 2).balance_loss.backward()
    first = x.grad.clone()
    r = Q.route_forward(x.detach(), 2)
    assert torch.equal(first, Q.route_backward(None, torch.ones((), device=DEV), r))
    x.grad = None
    Q.route(x, 2).weights.sum().backward()
    assert x.grad.abs().max() < 1e-6


def test_group_offsets():
    counts = torch.tensor([3, 0, 5], dtype=torch.int32, device=DEV)
    got = Q.group_offsets(counts)
    assert got.dtype == torch.int32 and got.tolist() == [0, 3, 3, 8]


def test_refusals():
    x = torch.zeros(4, 8, device=DEV)
    r = Q.route_forward(x, 2)
    for bad in (0, 9, -1):
        with pytest.raises(ValueError):
            Q.route_forward(x, bad)
    with pytest.raises(ValueError):
        Q.route_forward(torch.zeros(2, 1025, device=DEV), 2)
    with pytest.raises(ValueError):
        Q.route_forward(torch.zeros(2, 64, device=DEV), 33)
    with pytest.raises(TypeError):
        Q.route_forward(x.double(), 2)
    with pytest.raises(RuntimeError):
        Q.route_forward(x.cpu(), 2)
    with pytest.raises(TypeError):
        Q.route_forward(x, 2, valid=torch.ones(4, device=DEV))
    with pytest.raises(ValueError):
        Q.route_forward(x, 2, valid=torch.ones(3, dtype=torch.bool, device=DEV))
    with pytest.raises(ValueError):
        Q.route_backward(torch.zeros(4, 3, device=DEV), None, r)
    with pytest.raises(TypeError):
        Q.route_backward(torch.zeros(4, 2, device=DEV).half(), None, r)
    with pytest.raises(ValueError):
        Q.route_backward(None, torch.zeros(2, device=DEV), r)


def test_gradient_of_a_missing_choice_is_ignored():
    logits = _logits(5, 8, torch.float32)
    logits[2, 1:] = -math.inf                             # one expert for three choices
    dw = torch.ones(5, 3)
    dw[2, 1:] = math.nan
    for renormalize in (True, False):
        r = Q.route_forward(logits.to(DEV), 3, renormalize=renormalize)
        dl = Q.route_backward(dw.to(DEV), None, r)
        assert r.experts[2].tolist() == [0, -1, -1] and torch.isfinite(dl).all()


@pytest.mark.parametrize("experts", [8, 16, 32, 64, 100, 128, 256, 512, 1024])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=_ids)
def test_order_of_every_16_bit_pattern(dtype, experts):
    # both zeros, every payload and sign of a NaN, infinities and subnormal numbers
    g = torch.Generator().manual_seed(experts)
    bits = torch.randperm(65536, generator=g)[: 65536 // experts * experts]
    logits = (bits - 32768).to(torch.int16).view(dtype).view(-1, experts)
    k = min(experts, 32)
    order = logits.double()
    order[order == math.inf] = 1e300
    order[order.isnan()] = math.inf
    order, want = order.sort(dim=-1, descending=True, stable=True)
    want[order == -math.inf] = -1
    got = Q.route_forward(logits.to(DEV), k).experts.cpu()
    assert torch.equal(got.long(), want[:, :k])


@pytest.mark.parametrize("experts,k", [(64, 8), (128, 10), (200, 12), (256, 32), (512, 3)])
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_more_rows_than_the_blocks_hold(dtype, experts, k):
    # the wide blocks, several rounds of rows in each; choices against a sort, counts against the choices
    rows = 40009
    logits = torch.randn(rows, experts, generator=torch.Generator(DEV).manual_seed(k), device=DEV).to(dtype)
    valid = torch.ones(rows, dtype=torch.bool, device=DEV)
    valid[5::7] = False
    r = Q.route_forward(logits, k, valid=valid)
    want = logits.double().sort(dim=-1, descending=True, stable=True).indices[:, :k]
    want[5::7] = -1
    assert torch.equal(r.experts.long(), want)
    assert torch.equal(r.counts.long(), torch.bincount(want[want >= 0], minlength=experts))
    p = torch.softmax(logits.double(), -1)
    w = p.gather(-1, want.clamp(min=0))
    w = torch.where(want >= 0, w / w.sum(-1, keepdim=True), 0.0)
    # a probability is (2 (4 + |l - max|) + experts) 2^-24 off, as above; |l| < 8
    one = (2 * (4 + 16) + experts) * EPS32
    assert ((r.weights.double() - w).abs() <= 2 * one * w).all()
    n = valid.sum().double()
    balance = (experts * r.counts.double() / (k * n) * p[valid].sum(0) / n).sum().item()
    assert abs(r.balance_loss.item() - balance) <= (one + (rows + experts + 8) * EPS32) * balance
