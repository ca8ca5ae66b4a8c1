"""Expert router: softmax, top-k, per-expert counts and the balance loss, with gradients.

For the logits l of a token over E experts, p = softmax(l).  The k largest logits are chosen, ties to
the lowest index; the weight of a choice is its p, divided by the sum of the chosen p where
``renormalize``.  Over the n tokens that are valid

    balance_loss = sum_e (E counts_e / (k n)) (mean of p_e)

which is 1 for an even router and up to E for one that sends every token to the same expert;
gradients flow through the mean of p, the counts are constants.  -inf masks an expert: it is never
chosen.  A token that is not valid, or whose logits are all -inf, has choices -1 and weights 0, counts
nowhere and gets no gradient.

``route`` is differentiable; ``route_forward`` and ``route_backward`` are the calls below it.  ``counts``
gives the offsets of ``activations.grouped_linear`` by a running sum (``group_offsets``).
"""

from __future__ import annotations

import functools
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as N
from .activations import _dtype_code, _rows_of, _same

__all__ = ["Routed", "Routing", "route", "route_forward", "route_backward", "group_offsets"]

MAX_EXPERTS, MAX_K = 1024, 32


class Routed(NamedTuple):
    """weights float32 [..., k], experts int32 [..., k] (-1: no choice), counts int32 [E], balance_loss float32."""
    weights: torch.Tensor
    experts: torch.Tensor
    counts: torch.Tensor
    balance_loss: torch.Tensor


class Routing(NamedTuple):
    """The outputs of ``route_forward`` and what its backward call reads: the logits as they were, and
    ``stats``, two float32 for each token (its largest logit, 1 / sum exp), the number of valid tokens
    behind them."""
    weights: torch.Tensor
    experts: torch.Tensor
    counts: torch.Tensor
    balance_loss: torch.Tensor
    logits: torch.Tensor
    stats: torch.Tensor
    k: int
    renormalize: bool


@functools.lru_cache(maxsize=1024)
def _workspace(rows: int, experts: int, device: int) -> int:
    return int(N.lib().aw4_route_forward_workspace(rows, experts, device))


def route_forward(logits: torch.Tensor, k: int, valid: torch.Tensor | None = None,
                  renormalize: bool = True) -> Routing:
    """Routes tokens with logits [..., E] (float32, bfloat16 or float16; E up to 1024, k up to 32).
    ``valid``: bool [...], false for padding."""
    code = _dtype_code(logits, "route")
    src, rows, experts, ld = _rows_of(logits, "route")
    if experts < 1 or experts > MAX_EXPERTS:
        raise ValueError(f"route: 1 to {MAX_EXPERTS} experts expected, found {experts}")
    if not 1 <= k <= min(experts, MAX_K):
        raise ValueError(f"route: k from 1 to {min(experts, MAX_K)} expected, found {k}")
    dev, lead = logits.get_device(), logits.shape[:-1]
    if valid is not None:
        _same(valid, logits.device, torch.bool, "route: valid")
        if valid.shape != lead:
            raise ValueError(f"route: valid of shape {tuple(lead)} expected, found {tuple(valid.shape)}")
        valid = valid.contiguous()
    weights = logits.new_empty((*lead, k), dtype=torch.float32)
    chosen = logits.new_empty((*lead, k), dtype=torch.int32)
    counts = chosen.new_empty(experts)
    balance = weights.new_empty(())
    nbytes = _workspace(rows, experts, dev)
    # statistics, the number of valid rows, and behind them the call's workspace
    stats = weights.new_empty(2 * rows + 2 + nbytes // 4)
    at = stats.data_ptr()
    N.check(N.lib().aw4_route_forward(src.data_ptr(), code, rows, experts, ld, k, N.ptr(valid), int(renormalize),
                                      weights.data_ptr(), chosen.data_ptr(), at, counts.data_ptr(), at + 8 * rows,
                                      balance.data_ptr(), at + 8 * rows + 8, nbytes, dev, N.stream_of(dev)),
            "aw4_route_forward")
    return Routing(weights, chosen, counts, balance, logits, stats, k, renormalize)


def route_backward(dweights: torch.Tensor | None, dbalance: torch.Tensor | None,
                   routing: Routing) -> torch.Tensor:
    """The gradient of the logits from those of the weights ([..., k], float32) and of the balance loss (a
    float32 scalar on the device); None is zero."""
    logits = routing.logits
    src, rows, experts, ld = _rows_of(logits, "route_backward")
    dev = logits.device
    index = logits.get_device()
    if dweights is not None:
        _same(dweights, dev, torch.float32, "route_backward: dweights")
        if dweights.shape != routing.weights.shape:
            raise ValueError(f"route_backward: dweights of shape {tuple(routing.weights.shape)} expected, "
                             f"found {tuple(dweights.shape)}")
        dweights = dweights.contiguous()
    if dbalance is not None:
        _same(dbalance, dev, torch.float32, "route_backward: dbalance")
        if dbalance.numel() != 1:
            raise ValueError(f"route_backward: a scalar dbalance expected, found {tuple(dbalance.shape)}")
    dlogits = logits.new_empty(logits.shape)
    N.check(N.lib().aw4_route_backward(src.data_ptr(), N.DTYPE_CODES[logits.dtype], rows, experts, ld, routing.k,
                                       int(routing.renormalize), routing.weights.data_ptr(),
                                       routing.experts.data_ptr(), routing.stats.data_ptr(),
                                       routing.counts.data_ptr(), routing.stats.data_ptr() + 8 * rows,
                                       N.ptr(dweights), N.ptr(dbalance),
                                       dlogits.data_ptr(), index, N.stream_of(index)), "aw4_route_backward")
    return dlogits


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, valid, renormalize):
        r = route_forward(logits, k, valid, renormalize)
        ctx.save_for_backward(r.weights, r.experts, r.counts, logits, r.stats)
        ctx.k, ctx.renormalize = k, renormalize
        ctx.mark_non_differentiable(r.experts, r.counts)
        ctx.set_materialize_grads(False)
        return r.weights, r.experts, r.counts, r.balance_loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, _experts, _counts, dbalance):
        weights, experts, counts, logits, stats = ctx.saved_tensors
        r = Routing(weights, experts, counts, None, logits, stats, ctx.k, ctx.renormalize)
        return route_backward(dweights, dbalance, r), None, None, None


def route(logits: torch.Tensor, k: int, valid: torch.Tensor | None = None, renormalize: bool = True) -> Routed:
    """Differentiable router; see the module's head."""
    return Routed(*_Route.apply(logits, k, valid, renormalize))


def group_offsets(counts: torch.Tensor) -> torch.Tensor:
    """Offsets int32 [E + 1] of groups of these sizes, laid end to end."""
    if counts.dim() != 1:
        raise ValueError(f"group_offsets: one count for each expert expected, found {tuple(counts.shape)}")
    out = torch.zeros(counts.numel() + 1, dtype=torch.int32, device=counts.device)
    torch.cumsum(counts, 0, dtype=torch.int32, out=out[1:])
    return out
