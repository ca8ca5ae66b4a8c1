"""8-bit activation checkpoints and their use in the backward pass, against 64-bit definitions.

Tolerances: codes, exponents and read-back values are exact.  A computed value may be off by its
rounding to the dtype (UNIT, half a unit in the last place, and STEP near zero) plus the float32
evaluation: a handful of roundings of 2^-24 each on the terms' magnitudes, and for a sum of n terms at
most n of them (a tensor core that truncates loses up to twice that).
"""

from __future__ import annotations

import math

import pytest
import torch

from adamw4bit_b200 import activations as A
from tests import act8_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS32 = 2.0 ** -24


def _ids(v):
    return str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None


def _randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    size = torch.exp(torch.randn(shape[-1], generator=g)) * scale
    return (torch.randn(*shape, generator=g) * size).to(dtype)


def _close(got, ref, dtype, slack):
    """|got - ref| <= rounding of ref to dtype + slack, elementwise; not-a-numbers in the same places."""
    got = got.detach().cpu().double()
    assert got.shape == ref.shape
    bad = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), bad)
    tol = (1 + 2 ** -6) * R.UNIT[dtype] * ref.abs() + R.STEP[dtype] + slack
    off = ((got - ref).abs() - tol)[~bad]
    assert off.numel() == 0 or off.max() <= 0, f"off by {off.max().item():.3g} more than allowed"


def _edge_rows(dtype):
    """Rows of 96 values with what a checkpoint can meet: zeros, ties, the dtype's extremes and
    smallest steps, infinities and NaN."""
    big, step = torch.finfo(dtype).max, R.STEP[dtype]
    x = torch.zeros(12, 96)
    x[1] = torch.linspace(-1, 1, 96)
    x[2, ::2], x[2, 1::2] = 127.0, 0.5                   # ties at half a step
    x[3, :3] = torch.tensor([127.5, 1.5, -2.5])
    x[4, 5], x[4, 40], x[4, 70] = big, -big, big / 2
    x[5, 3], x[5, 33] = step, -3 * step
    x[6, 10], x[6, 11], x[6, 50], x[6, 80] = math.inf, 1.0, -math.inf, 7.0
    x[7, 31], x[7, 32] = math.nan, 3.0
    x[8] = torch.finfo(dtype).min
    x[9, 64] = torch.finfo(dtype).tiny
    x[10] = 63.99
    x[11] = -127.49
    return x.to(dtype)


SHAPES = [(1, 1), (1, 31), (1, 32), (3, 33), (5, 8), (7, 1001), (64, 768), (300, 72), (2, 3, 40), (130, 4100),
          (1000,), (33, 1024)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_checkpoint_is_exact(dtype, shape):
    x = _randn(*shape, dtype=dtype)
    c = A.quantize_act8(x.to(DEV))
    flat = x.reshape(-1, shape[-1])
    codes, scales = R.encode(flat)
    assert torch.equal(c.codes.cpu().long(), codes)
    assert torch.equal(c.scales.cpu().long(), scales)
    back = c.dequantize()
    assert back.dtype == dtype and back.shape == x.shape
    assert torch.equal(back.cpu().double().reshape(flat.shape), R.decode(codes, scales, shape[-1]))
    assert c.nbytes == scales.numel() * 33


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_checkpoint_edge_values(dtype):
    x = _edge_rows(dtype)
    c = A.quantize_act8(x.to(DEV))
    codes, scales = R.encode(x)
    assert torch.equal(c.scales.cpu().long(), scales)
    fine = (scales != 255).repeat_interleave(32, 1)
    assert torch.equal(c.codes.cpu().long()[fine], codes[fine])
    ref, got = R.decode(codes, scales, 96), c.dequantize().cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(got.nan_to_num(0.0), ref.nan_to_num(0.0))


@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_checkpoint_strides(dtype):
    base = _randn(40, 200, dtype=dtype).to(DEV)
    for x in (base[:, 3:100], base[::2, 8:72], base.t(), base[:1].expand(5, 200), base.view(4, 10, 200)[:, 2:7],
              base[:, 5:6], base.view(4, 10, 200).transpose(0, 1)):
        want = R.values(x.cpu().reshape(-1, x.shape[-1])).reshape(x.shape)
        assert torch.equal(A.quantize_act8(x).dequantize().cpu().double(), want)


@pytest.mark.parametrize("shape", [(0, 64), (4, 0), (0, 0)], ids=str)
def test_empty(shape):
    x = torch.empty(shape, dtype=torch.bfloat16, device=DEV)
    assert A.quantize_act8(x).dequantize().shape == shape
    w = torch.ones(shape[1], dtype=torch.bfloat16, device=DEV)
    y, saved = A.rms_norm_forward(x, w)
    dx, dw = A.rms_norm_backward(x, w, saved)
    assert y.shape == dx.shape == shape and torch.equal(dw, torch.zeros_like(w))
    h, saved = A.swiglu_forward(x, x)
    assert h.shape == shape and A.swiglu_backward(h, saved)[1].shape == shape
    dy = torch.empty(shape[0], 24, dtype=torch.bfloat16, device=DEV)
    dw = A.weight_grad(dy, A.quantize_act8(x))
    assert dw.shape == (24, shape[1]) and not dw.any()


def test_more_than_2_31_values():
    rows, cols = 65600, 32768
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    x[-3:] = _randn(3, cols, dtype=torch.bfloat16).to(DEV)
    x[0, :64] = 2.0
    c = A.quantize_act8(x)
    back = c.dequantize()
    assert torch.equal(back[-3:].cpu().double(), R.values(x[-3:].cpu()))
    assert torch.equal(back[:1], x[:1]) and not back[1:-3].any()
    del back
    dw = A.weight_grad(x[:, :8], c)
    want, mag = R.weight_grad(x[-3:, :8].cpu(), R.values(x[-3:].cpu()))
    want[:, :64] += 4.0 * (torch.arange(8) < 8)[:, None]
    mag[:, :64] += 4.0
    _close(dw, want, torch.bfloat16, 8 * EPS32 * mag)


# ---------------------------------------------------------------------------
# RMS norm
# ---------------------------------------------------------------------------

NORM_SHAPES = [(1, 1), (1, 768), (5, 33), (64, 256), (513, 64), (37, 1000), (9, 1531), (3, 2050), (700, 2048),
               (4, 4096), (3, 8191), (2, 16384), (2, 5, 96),
               (1001, 128), (333, 24), (40000, 64), (130, 1280), (70, 2560), (40, 5120), (30, 6144), (20, 7168), (10, 12288)]


def _check_norm(x, w, dy, y, saved, dx, dw, eps):
    flat, dflat = x.reshape(-1, x.shape[-1]), dy.reshape(-1, x.shape[-1])
    rows, cols = flat.shape
    ref, r = R.rms_norm(flat, w, eps)
    # the sum of squares is off by at most cols roundings (cols / 2 of them reach r), the rest a few
    few = (cols / 2 + 8) * EPS32
    _close(y.reshape(flat.shape), ref, x.dtype, few * ref.abs())
    v = R.values(flat)
    assert torch.equal(saved.x8.dequantize().cpu().double().reshape(flat.shape), v)
    gx, mx, gw, mw = R.rms_norm_backward(dflat, w, v, r)
    _close(dx.reshape(flat.shape), gx, x.dtype, (3 * few + cols * EPS32) * mx)
    _close(dw, gw, w.dtype, (few + (rows + 4) * EPS32) * mw)


@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                          (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                          (torch.float16, torch.float32)], ids=_ids)
def test_rms_norm(dtype, wdtype, shape):
    x, dy = _randn(*shape, dtype=dtype), _randn(*shape, seed=1, dtype=dtype, scale=0.1)
    w = (1 + 0.3 * _randn(shape[-1], seed=2)).to(wdtype)
    if len(shape) == 2 and shape[0] > 4:
        x[2] = 0
    y, saved = A.rms_norm_forward(x.to(DEV), w.to(DEV), 1e-5)
    dx, dw = A.rms_norm_backward(dy.to(DEV), w.to(DEV), saved)
    assert dw.dtype == wdtype
    _check_norm(x, w, dy, y, saved, dx, dw, 1e-5)


def test_rms_norm_strides_and_output_checkpoint():
    base = _randn(24, 300, dtype=torch.bfloat16).to(DEV)
    w = (1 + 0.3 * _randn(130, seed=2)).to(torch.bfloat16).to(DEV)
    for x in (base[:, 5:135], base[::3, 8:138]):
        dy = base.flip(0)[: x.shape[0], 100:230]
        y, saved = A.rms_norm_forward(x, w, 1e-5, checkpoint_output=True)
        dx, dw = A.rms_norm_backward(dy, w, saved)
        _check_norm(x.cpu(), w.cpu(), dy.cpu(), y, saved, dx, dw, 1e-5)
        assert torch.equal(saved.output.dequantize().cpu().double(), R.values(y.cpu()))


@pytest.mark.parametrize("cols", [96, 1100, 5000])
def test_rms_norm_bad_row_stays_in_its_row(cols):
    x, dy = _randn(6, cols), _randn(6, cols, seed=1)
    w = torch.ones(cols)
    x[3, 40] = math.inf
    x[4, 1] = math.nan
    y, saved = A.rms_norm_forward(x.to(DEV), w.to(DEV))
    dx, dw = A.rms_norm_backward(dy.to(DEV), w.to(DEV), saved)
    good = [0, 1, 2, 5]
    ref, r = R.rms_norm(x[good], w, 1e-6)
    _close(y[good], ref, x.dtype, (cols / 2 + 8) * EPS32 * ref.abs())
    gx, mx, _, _ = R.rms_norm_backward(dy[good], w, R.values(x[good]), r)
    _close(dx[good], gx, x.dtype, (3 * cols + 24) * EPS32 * mx)
    assert torch.isnan(y[4]).all() and torch.isnan(dx[4]).all() and torch.isnan(dw).any()


# ---------------------------------------------------------------------------
# gated activation
# ---------------------------------------------------------------------------

def _check_swiglu(g, u, dh, h, saved, dg, du):
    flat = lambda t: t.reshape(-1, g.shape[-1])  # noqa: E731
    g, u, dh = flat(g), flat(u), flat(dh)
    # the argument of the exponential rounds by |g| 2^-23, its value by a few units of 2^-22
    few = (16 + 4 * g.double().abs()) * EPS32
    ref = R.swiglu(g, u)
    _close(flat(h), ref, g.dtype, few * ref.abs() + 1e-37)
    v, w = R.values(g), R.values(u)
    assert torch.equal(flat(saved.gate8.dequantize()).cpu().double(), v)
    assert torch.equal(flat(saved.up8.dequantize()).cpu().double(), w)
    few = (16 + 4 * v.abs()) * EPS32
    a, b = R.swiglu_backward(dh, v, w)
    s = torch.sigmoid(v)
    # 1 - s loses what s has lost, in units of s
    mag = (dh.double() * w * s).abs() * (1 + v.abs())
    _close(flat(dg), a, g.dtype, few * mag + 1e-37)
    _close(flat(du), b, g.dtype, few * b.abs() + 1e-37)


@pytest.mark.parametrize("shape", [(1, 1), (3, 33), (37, 1001), (64, 768), (2, 3, 40), (9, 5632)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_swiglu(dtype, shape):
    g, u, dh = (_randn(*shape, seed=s, dtype=dtype) for s in (0, 1, 2))
    h, saved = A.swiglu_forward(g.to(DEV), u.to(DEV))
    dg, du = A.swiglu_backward(dh.to(DEV), saved)
    _check_swiglu(g, u, dh, h, saved, dg, du)


@pytest.mark.parametrize("cols", [1, 31, 64, 1001])
@pytest.mark.parametrize("dtype", DTYPES, ids=_ids)
def test_swiglu_packed_and_strided(dtype, cols):
    both, dh = _randn(19, 2 * cols, dtype=dtype), _randn(19, cols, seed=3, dtype=dtype)
    h, saved = A.swiglu_forward(both.to(DEV), checkpoint_output=True)
    out = A.swiglu_backward(dh.to(DEV), saved)
    assert out.shape == both.shape
    _check_swiglu(both[:, :cols], both[:, cols:], dh, h, saved, out[:, :cols], out[:, cols:])
    assert torch.equal(saved.output.dequantize().cpu().double(), R.values(h.cpu()))
    wide = _randn(40, 3 * cols + 5, dtype=dtype).to(DEV)
    g, u, d = wide[::2, 1:1 + cols], wide[1::2, 2:2 + cols], wide[:1, :cols].expand(20, cols)
    h, saved = A.swiglu_forward(g, u)
    _check_swiglu(g.cpu(), u.cpu(), d.cpu(), h, saved, *A.swiglu_backward(d, saved))


def test_swiglu_extremes():
    g = torch.tensor([[-200.0, -90.0, -1e30, 200.0, 1e30, 0.0, -0.0, 5.0] * 4])
    u, dh = torch.full_like(g, 2.0), torch.ones_like(g)
    h, saved = A.swiglu_forward(g.to(DEV), u.to(DEV))
    _close(h, R.swiglu(g, u), g.dtype, 1e-30 + 1e-5 * R.swiglu(g, u).abs())
    dg, du = A.swiglu_backward(dh.to(DEV), saved)
    assert torch.isfinite(dg).all() and torch.isfinite(du).all()


# ---------------------------------------------------------------------------
# weight gradient
# ---------------------------------------------------------------------------

def _check_wgrad(dw, dy, x, offsets=None, start=None, rows=None):
    ref, mag = R.weight_grad(dy, R.values(x), offsets)
    rows = rows or max(1, dy.shape[0])
    if start is not None:
        ref, mag = ref + start.double(), mag + start.double().abs()
    _close(dw, ref, dw.dtype, 2 * (rows + 2) * EPS32 * mag)


WGRAD = [(1, 8, 32), (16, 64, 64), (63, 8, 40), (65, 128, 256), (64, 130, 100), (200, 257, 264), (1000, 24, 33),
         (129, 7, 1), (500, 1, 500), (300, 768, 768), (4096, 64, 96), (96, 1000, 2050),
         (200, 600, 411), (70, 520, 412)]


@pytest.mark.parametrize("rows,n,k", WGRAD)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=_ids)
def test_weight_grad(dtype, rows, n, k):
    x, dy = _randn(rows, k, dtype=dtype), _randn(rows, n, seed=1, dtype=dtype, scale=0.1)
    x8 = A.quantize_act8(x.to(DEV))
    dw = A.weight_grad(dy.to(DEV), x8)
    assert dw.dtype == dtype and dw.shape == (n, k)
    _check_wgrad(dw, dy, x)
    again = A.weight_grad(dy.to(DEV), x8)
    assert torch.equal(dw.view(torch.int16), again.view(torch.int16))
    start = _randn(n, k, seed=5)
    total = start.to(DEV)
    assert A.weight_grad(dy.to(DEV), x8, out=total, accumulate=True) is total
    _check_wgrad(total, dy, x, start=start)
    _check_wgrad(A.weight_grad(dy.to(DEV), x8, out_dtype=torch.float32), dy, x)


@pytest.mark.parametrize("counts", [[0, 0, 0], [5], [1, 0, 64, 63, 65, 0], [700, 3, 128, 200], [0, 33] * 20],
                         ids=lambda c: "-".join(map(str, c[:6])))
@pytest.mark.parametrize("n,k", [(64, 96), (136, 300), (13, 7), (512, 1024)])
def test_weight_grad_groups(n, k, counts):
    rows = sum(counts)
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    x, dy = _randn(rows, k, dtype=torch.bfloat16), _randn(rows, n, seed=1, dtype=torch.bfloat16)
    off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    x8 = A.quantize_act8(x.to(DEV))
    dw = A.weight_grad(dy.to(DEV), x8, off)
    assert dw.shape == (len(counts), n, k)
    _check_wgrad(dw, dy, x, offsets)
    start = _randn(len(counts), n, k, seed=4).to(torch.bfloat16)
    total = start.to(DEV)
    A.weight_grad(dy.to(DEV), x8, off, out=total, accumulate=True)
    _check_wgrad(total, dy, x, offsets, start=start)


@pytest.mark.parametrize("n,k,counts", [(600, 300, [4000, 10, 0, 100]),      # one long group: its tiles are cut
                                        (130, 520, [0, 65, 2500, 1, 1900, 0]),
                                        (5000, 4000, [2000])])               # whole rounds and cut tiles
def test_weight_grad_cut_tiles(n, k, counts):
    rows, offsets = sum(counts), [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    x, dy = _randn(rows, k, dtype=torch.bfloat16), _randn(rows, n, seed=1, dtype=torch.bfloat16)
    x8 = A.quantize_act8(x.to(DEV))
    off = torch.tensor(offsets, dtype=torch.int32, device=DEV) if len(counts) > 1 else None
    dw = A.weight_grad(dy.to(DEV), x8, off)
    _check_wgrad(dw, dy, x, offsets if len(counts) > 1 else None)
    again = A.weight_grad(dy.to(DEV), x8, off)
    assert torch.equal(dw.view(torch.int16), again.view(torch.int16))
    total = torch.ones_like(dw, dtype=torch.float32)
    A.weight_grad(dy.to(DEV), x8, off, out=total, accumulate=True)
    _check_wgrad(total, dy, x, offsets if len(counts) > 1 else None, start=torch.ones(total.shape))


def test_weight_grad_bad_rows_stay_in_their_group():
    counts = [30, 50, 20, 100]
    offsets = [0, 30, 80, 100, 200]
    x, dy = _randn(200, 96, dtype=torch.bfloat16), _randn(200, 72, seed=1, dtype=torch.bfloat16)
    x[30, 3], x[79, 50] = math.nan, math.inf
    dy[31, 5], dy[78, 6] = math.inf, math.nan
    dw = A.weight_grad(dy.to(DEV), A.quantize_act8(x.to(DEV)), torch.tensor(offsets, dtype=torch.int32, device=DEV))
    for g in (0, 2, 3):
        a, b = offsets[g], offsets[g + 1]
        _check_wgrad(dw[g], dy[a:b], x[a:b])
    assert torch.isnan(dw[1]).any() and len(counts) == dw.shape[0]


def test_weight_grad_offsets_are_cut_to_the_rows():
    x, dy = _randn(70, 64, dtype=torch.bfloat16), _randn(70, 40, seed=1, dtype=torch.bfloat16)
    off = torch.tensor([-5, 20, 10, 90, 200], dtype=torch.int32, device=DEV)
    dw = A.weight_grad(dy.to(DEV), A.quantize_act8(x.to(DEV)), off)
    _check_wgrad(dw[0], dy[:20], x[:20])
    assert not dw[1].any() and not dw[3].any()
    _check_wgrad(dw[2], dy[10:], x[10:])


@pytest.mark.parametrize("lo,hi", [(0, 64), (8, 72), (3, 67), (1, 130)])
def test_weight_grad_strides(lo, hi):
    base = _randn(150, 200, dtype=torch.float16).to(DEV)
    x = _randn(75, 130, seed=2, dtype=torch.float16)
    x8 = A.quantize_act8(x.to(DEV))
    for dy in (base[::2, lo:hi], base[:75, lo:hi], base[:1, lo:hi].expand(75, hi - lo), base[lo:hi, :75].t()):
        _check_wgrad(A.weight_grad(dy, x8), dy.cpu(), x)


# ---------------------------------------------------------------------------
# gradients, streams, graphs
# ---------------------------------------------------------------------------

def _on_grid(*shape, seed):
    """Values that their checkpoint holds exactly: k / 64, each block with one of size 1 or more."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-127, 128, shape, generator=g).float() / 64
    x[..., ::32] = 1.5
    return x


def _difference(f, inputs, directions, h):
    up = f(*[x + h * d for x, d in zip(inputs, directions)])
    down = f(*[x - h * d for x, d in zip(inputs, directions)])
    return (up - down) / (2 * h)


@pytest.mark.parametrize("op", ["rms_norm", "swiglu", "swiglu_packed"])
def test_gradient_against_differences(op):
    a, b, c = _on_grid(6, 96, seed=1), _on_grid(6, 96, seed=2), _randn(6, 96, seed=3, scale=0.1)
    if op == "rms_norm":
        b = _on_grid(96, seed=4)
        own = lambda x, w: A.rms_norm(x, w, 1e-5)  # noqa: E731
        ref = lambda x, w: (R.rms_norm(x, w, 1e-5)[0] * c.double()).sum()  # noqa: E731
    elif op == "swiglu":
        own, ref = A.swiglu, lambda g, u: (R.swiglu(g, u) * c.double()).sum()
    else:
        own = lambda g, u: A.swiglu(torch.cat([g, u], -1))  # noqa: E731
        ref = lambda g, u: (R.swiglu(g, u) * c.double()).sum()  # noqa: E731
    x = [t.to(DEV).requires_grad_() for t in (a, b)]
    (own(*x) * c.to(DEV)).sum().backward()
    for i in range(2):
        d = [torch.zeros_like(a).double(), torch.zeros_like(b).double()]
        d[i] = _randn(*d[i].shape, seed=7 + i).double()
        want = _difference(ref, [a.double(), b.double()], d, 1e-5)
        terms = x[i].grad.cpu().double() * d[i]
        # central differences: h^2 times a third derivative (values of order 10), float64 cancellation
        # 1e-16 / 1e-5; the gradient itself float32
        assert abs(terms.sum() - want) <= 1e-8 * 96 * 6 + 300 * EPS32 * terms.abs().sum()


def test_linear_and_grouped_linear_gradients():
    x = _on_grid(50, 64, seed=1).to(torch.bfloat16)
    w = _randn(3, 40, 64, seed=2, scale=0.1).to(torch.bfloat16)
    c = _randn(50, 40, seed=3).to(torch.bfloat16)
    bias = _randn(40, seed=4).to(torch.bfloat16)
    xs, ws, bs = (t.to(DEV).requires_grad_() for t in (x, w[0], bias))
    y = A.linear(xs, ws, bs)
    y.backward(c.to(DEV))
    cd, xd = c.double(), x.double()
    _close(y, xd @ w[0].double().t() + bias.double(), torch.bfloat16, 0.01)
    _close(xs.grad, cd @ w[0].double(), torch.bfloat16, 64 * 2 * EPS32 * (cd.abs() @ w[0].double().abs()))
    _close(ws.grad, cd.t() @ xd, torch.bfloat16, 2 * 52 * EPS32 * (cd.abs().t() @ xd.abs()))
    _close(bs.grad, cd.sum(0), torch.bfloat16, 52 * EPS32 * cd.abs().sum(0))
    offsets = torch.tensor([0, 17, 17, 50], dtype=torch.int32, device=DEV)
    xs, ws = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    y = A.grouped_linear(xs, ws, offsets)
    y.backward(c.to(DEV))
    for g, (a, b) in enumerate(((0, 17), (17, 17), (17, 50))):
        _close(y[a:b], xd[a:b] @ w[g].double().t(), torch.bfloat16, 0.01)
        _close(xs.grad[a:b], cd[a:b] @ w[g].double(), torch.bfloat16,
               64 * 2 * EPS32 * (cd[a:b].abs() @ w[g].double().abs()))
        _close(ws.grad[g], cd[a:b].t() @ xd[a:b], torch.bfloat16, 2 * 52 * EPS32 * (cd[a:b].abs().t() @ xd[a:b].abs()))


def test_linear_keeps_a_given_checkpoint():
    x = _randn(33, 96, dtype=torch.bfloat16).to(DEV).requires_grad_()
    nw = torch.ones(96, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    w = _randn(24, 96, seed=2, dtype=torch.bfloat16).to(DEV).requires_grad_()
    y, y8 = A.rms_norm(x, nw, checkpoint_output=True)
    A.linear(y, w, x8=y8).sum().backward()
    first = [t.grad.clone() for t in (x, nw, w)]
    for t in (x, nw, w):
        t.grad = None
    A.linear(A.rms_norm(x, nw), w).sum().backward()
    assert all(torch.equal(a, t.grad) for a, t in zip(first, (x, nw, w)))
    g = _randn(33, 96, seed=6, dtype=torch.bfloat16).to(DEV).requires_grad_()
    h, h8 = A.swiglu(g, x, checkpoint_output=True)
    A.linear(h, w, x8=h8).sum().backward()
    assert torch.isfinite(g.grad).all()


def test_runs_on_the_current_stream_and_in_a_graph():
    x = _randn(64, 256, dtype=torch.bfloat16).to(DEV)
    dy = _randn(64, 128, seed=1, dtype=torch.bfloat16).to(DEV)
    want = A.weight_grad(dy, A.quantize_act8(x))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        hold = torch.zeros(1 << 26, device=DEV)
        for _ in range(8):
            hold.add_(1.0)                        # work ahead of the copy on the side stream
        late = x.clone()
        got = A.weight_grad(dy, A.quantize_act8(late))
    side.synchronize()
    assert torch.equal(got, want)
    xs = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = A.weight_grad(dy, A.quantize_act8(xs))
    xs.zero_()
    graph.replay()
    assert not out.any()
    xs.copy_(x)
    graph.replay()
    assert torch.equal(out, want)


def test_refusals():
    x = torch.ones(4, 64, device=DEV, dtype=torch.bfloat16)
    x8 = A.quantize_act8(x)
    w = torch.ones(64, device=DEV, dtype=torch.bfloat16)
    y, saved = A.rms_norm_forward(x, w)
    off = torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    with pytest.raises(TypeError):
        A.quantize_act8(x.double())
    with pytest.raises(ValueError):
        A.quantize_act8(x[0, 0])
    with pytest.raises(RuntimeError):
        A.quantize_act8(x.cpu())
    with pytest.raises(ValueError):
        A.rms_norm_forward(x, w[:32])
    with pytest.raises(TypeError):
        A.rms_norm_forward(x, w.half())
    with pytest.raises(RuntimeError):
        A.rms_norm_forward(x, w.cpu())
    with pytest.raises(RuntimeError, match="16384"):
        A.rms_norm_forward(torch.ones(1, 16385, device=DEV), torch.ones(16385, device=DEV))
    with pytest.raises(ValueError):
        A.rms_norm_backward(x[:2], w, saved)
    with pytest.raises(TypeError):
        A.rms_norm_backward(x.float(), w, saved)
    with pytest.raises(ValueError):
        A.swiglu_forward(x[:, :63])
    with pytest.raises(ValueError):
        A.swiglu_forward(x, x[:2])
    with pytest.raises(TypeError):
        A.swiglu_forward(x, x.half())
    with pytest.raises(TypeError):
        A.weight_grad(x.float(), x8)
    with pytest.raises(TypeError):
        A.weight_grad(x.half(), x8)
    with pytest.raises(ValueError):
        A.weight_grad(x[:3], x8)
    with pytest.raises(TypeError):
        A.weight_grad(x, x8, off.long())
    with pytest.raises(ValueError):
        A.weight_grad(x, x8, off[:1])
    with pytest.raises(ValueError):
        A.weight_grad(x, x8, accumulate=True)
    with pytest.raises(ValueError):
        A.weight_grad(x, x8, out=torch.empty(64, 65, device=DEV))
    with pytest.raises(TypeError):
        A.weight_grad(x, x8, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        A.linear(x, torch.ones(8, 32, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        A.linear(x.float(), torch.ones(8, 64, device=DEV))
    with pytest.raises(ValueError):
        A.linear(x, torch.ones(8, 64, device=DEV, dtype=torch.bfloat16), x8=A.quantize_act8(x[:2]))
    with pytest.raises(ValueError):
        A.grouped_linear(x, torch.ones(2, 8, 64, device=DEV, dtype=torch.bfloat16), off)
