"""The 8-bit activation checkpoint and the operators that read it, from their definitions in 64 bits.

Every function takes and returns torch tensors on the CPU; widths are float64.  Beside a result, a
function that sums returns the sum of the terms' magnitudes, from which the tests derive how far a
float32 sum may be off.
"""

from __future__ import annotations

import math

import torch

BLOCK = 32
# half a unit in the last place, relative: the rounding of a result to its dtype
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# the smallest step of the dtype: what a rounding near zero may lose
STEP = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def encode(x: torch.Tensor):
    """(codes int64 [rows, pitch], scale bytes int64 [rows, blocks]) of x [rows, cols]."""
    e_min = -24 if x.dtype == torch.float16 else -126
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    v = torch.zeros(rows, blocks * BLOCK, dtype=torch.float64)
    v[:, :cols] = x.double()
    v = v.view(rows, blocks, BLOCK)
    codes = torch.zeros(rows, blocks, BLOCK, dtype=torch.int64)
    scales = torch.zeros(rows, blocks, dtype=torch.int64)
    finite = torch.isfinite(v).all(-1)
    most = torch.where(finite, v.abs().amax(-1), torch.zeros(()).double())
    _, exp2 = torch.frexp(most)
    e = torch.where(most > 0, exp2 - 1 - 6, torch.full_like(exp2, e_min)).clamp(min=e_min)
    q = torch.round(torch.ldexp(torch.where(finite[..., None], v, 0.0), -e[..., None])).clamp(-127, 127)
    codes[:] = q.to(torch.int64)
    scales[:] = torch.where(finite, e.to(torch.int64) + 127, 255)
    return codes.view(rows, blocks * BLOCK), scales


def decode(codes: torch.Tensor, scales: torch.Tensor, cols: int) -> torch.Tensor:
    v = codes.view(scales.shape[0], scales.shape[1], BLOCK).double()
    v = torch.ldexp(v, (scales - 127)[..., None])
    v[scales == 255] = math.nan
    return v.reshape(scales.shape[0], scales.shape[1] * BLOCK)[:, :cols]


def values(x: torch.Tensor) -> torch.Tensor:
    return decode(*encode(x), x.shape[1])


def rms_norm(x, w, eps):
    """(y, r)"""
    x, w = x.double(), w.double()
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * r * w, r


def rms_norm_backward(dy, w, v, r):
    """dx, magnitude of dx's terms, dw, magnitude of dw's terms"""
    dy, w = dy.double(), w.double()
    g = w * dy
    dx = r * g - v * r ** 3 * (v * g).mean(-1, keepdim=True)
    dx_mag = (r * g).abs() + v.abs() * r ** 3 * (v * g).abs().mean(-1, keepdim=True)
    return dx, dx_mag, (dy * v * r).sum(0), (dy * v * r).abs().sum(0)


def swiglu(g, u):
    g, u = g.double(), u.double()
    return g * torch.sigmoid(g) * u


def swiglu_backward(dh, g, u):
    dh = dh.double()
    s = torch.sigmoid(g)
    return dh * u * (s + g * s * (1 - s)), dh * g * s


def weight_grad(dy, v, offsets=None):
    """dW and the magnitude of its terms: [n, k], or [groups, n, k] with offsets."""
    dy = dy.double()
    bounds = [0, dy.shape[0]] if offsets is None else list(offsets)
    out = torch.stack([dy[a:b].t() @ v[a:b] for a, b in zip(bounds, bounds[1:])])
    mag = torch.stack([dy[a:b].abs().t() @ v[a:b].abs() for a, b in zip(bounds, bounds[1:])])
    return (out[0], mag[0]) if offsets is None else (out, mag)


def route(logits, k, valid=None, renormalize=True, dweights=None, dbalance=0.0):
    """weights, experts, counts, balance, dlogits of [rows, E], one row at a time."""
    l = logits.double()
    rows, experts = l.shape
    p = torch.zeros(rows, experts, dtype=torch.float64)
    weights = torch.zeros(rows, k, dtype=torch.float64)
    chosen = torch.full((rows, k), -1, dtype=torch.int64)
    counts = torch.zeros(experts, dtype=torch.int64)
    live = torch.zeros(rows, dtype=torch.bool)
    for t in range(rows):
        if (valid is not None and not bool(valid[t])) or bool((l[t] == -math.inf).all()):
            continue
        live[t] = True
        p[t] = torch.softmax(l[t], 0)
        rank = sorted(range(experts), key=lambda e: (0 if math.isnan(l[t, e]) else 1, -l[t, e].item(), e))
        for j, e in enumerate(rank[:k]):
            if l[t, e] == -math.inf:
                break
            chosen[t, j] = e
            weights[t, j] = p[t, e]
            counts[e] += 1
        if renormalize:
            weights[t] /= weights[t].sum()
    n = int(live.sum())
    if n == 0:
        return weights, chosen, counts, torch.zeros((), dtype=torch.float64), torch.zeros_like(p)
    share = experts * counts.double() / (k * n)
    balance = (share * p[live].sum(0) / n).sum()
    dl = torch.zeros_like(p)
    for t in range(rows):
        if not live[t]:
            continue
        dl[t] = p[t] * (share - (p[t] * share).sum()) * dbalance / n
        if dweights is None:
            continue
        at = [int(e) for e in chosen[t] if e >= 0]
        w, dw = weights[t, : len(at)], dweights[t, : len(at)].double()
        if not renormalize:
            dl[t] -= p[t] * (w * dw).sum()
            dl[t, at] += w * dw
        else:
            dl[t, at] += w * (dw - (w * dw).sum())
    return weights, chosen, counts, balance, dl
