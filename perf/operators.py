"""Cases of the 8-bit activation checkpoint operators and of the expert router.

A training step keeps two kinds of memory besides its weights: the optimizer's moments and the
activations that wait for the backward pass.  The operators here hold the second in 8 bits and run
the backward pass from that form; the router produces the per-expert counts that the grouped
weight gradient consumes, and the balance loss that keeps those counts even.

An activation's rows are cut into blocks of 32 values along the last axis.  A block keeps one
exponent e and 32 whole numbers q, |q| <= 127, and stands for q * 2^e:

    e = max(floor(log2(max |x|)) - 6, e_min)     e_min = -24 for float16, else -126
    q = clamp(round_half_even(x * 2^-e), -127, 127)

A block that holds an infinity or a NaN reads back as NaN.

    checkpoint   x -> (q, e) -> the values they stand for
    norm         y = x r w, r = (mean(x^2) + eps)^-1/2; backward from the checkpoint v of x:
                 dx = r (w dy) - v r^3 mean(v w dy), dw = sum over rows of dy v r
    swiglu       h = g sigmoid(g) u; backward from the checkpoints of g and u
    wgrad        dW_e = sum over the rows t of group e of dy_t v_t^T, v the checkpoint of x
    route        p = softmax(l); the k largest logits of a row (ties to the lowest index), their
                 p (divided by their sum where renormalized) as weights; counts per expert;
                 balance = E sum_e (counts_e / (k n)) mean over the n valid rows of p_e;
                 backward gives the gradient of the logits

Where ``own`` is false ``run`` is the plain form in elementary float32 operations, else the calls
of adamw4bit_b200.activations and adamw4bit_b200.routing.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-5
_BLOCK = 32


# ------------------------------------------------------------------------------------- cases

def listed():
    return [
        # the rows of a few tokens at the small model's width: launch latency
        {"name": "checkpoint_short", "op": "checkpoint", "rows": 16, "cols": 768, "dtype": "f32"},
        # the input of the 8B model's down projection, 8192 tokens: the largest single activation
        {"name": "checkpoint_ffn", "op": "checkpoint", "rows": 8192, "cols": 14336, "dtype": "bf16"},
        # one short sequence of the small model in float16, float32 norm weight
        {"name": "norm_short", "op": "norm", "rows": 64, "cols": 768, "dtype": "f16", "weight": "f32"},
        # a micro-batch of 16384 tokens of the 8B model
        {"name": "norm_long", "op": "norm", "rows": 16384, "cols": 4096, "dtype": "bf16", "weight": "bf16"},
        # an odd width in float32: rows that are not aligned to vectors, a ragged last block
        {"name": "norm_odd", "op": "norm", "rows": 2047, "cols": 1531, "dtype": "f32", "weight": "f32"},
        # a short, odd sequence, separate gate and up projections
        {"name": "swiglu_short", "op": "swiglu", "rows": 37, "cols": 1001, "dtype": "f16", "packed": False},
        # the 8B model's feed-forward over 8192 tokens, gate and up as halves of one projection
        {"name": "swiglu_ffn", "op": "swiglu", "rows": 8192, "cols": 14336, "dtype": "bf16", "packed": True},
        # one short sequence through a square projection of the small model
        {"name": "wgrad_short", "op": "wgrad", "rows": 96, "n": 768, "k": 768, "groups": 1, "dtype": "bf16"},
        # the up projection of the 8B model over 8192 tokens
        {"name": "wgrad_ffn", "op": "wgrad", "rows": 8192, "n": 14336, "k": 4096, "groups": 1, "dtype": "bf16"},
        # sixteen experts of the 1B model's feed-forward size, ragged, one of them without a token
        {"name": "wgrad_experts", "op": "wgrad", "rows": 16384, "n": 5632, "k": 2048, "groups": 16, "dtype": "f16"},
        # a short sequence over few experts, float32 logits
        {"name": "route_short", "op": "route", "rows": 48, "experts": 8, "k": 2, "dtype": "f32",
         "renormalize": True},
        # a global batch over many experts, one token in eight padding
        {"name": "route_long", "op": "route", "rows": 65536, "experts": 128, "k": 8, "dtype": "bf16",
         "renormalize": False},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A width over [low, high]: three in four a multiple of 32, as models have them."""
    v = _log(rng, low, high)
    return max(32, v // 32 * 32) if rng.random() < 0.75 and v >= 32 else v


def draw(rng):
    op = rng.choice(["checkpoint", "norm", "swiglu", "wgrad", "wgrad", "route"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "checkpoint":
        cols = _width(rng, 16, 14336)
        return {"op": op, "rows": _log(rng, 1, 8192), "cols": cols, "dtype": dtype}
    if op == "norm":
        return {"op": op, "rows": _log(rng, 1, 16384), "cols": _width(rng, 64, 4096), "dtype": dtype,
                "weight": rng.choice([dtype, "f32"])}
    if op == "swiglu":
        return {"op": op, "rows": _log(rng, 1, 8192), "cols": _width(rng, 16, 14336), "dtype": dtype,
                "packed": rng.random() < 0.5}
    if op == "wgrad":
        rows = _log(rng, 16, 16384)
        n = _width(rng, 64, 14336)
        k = _width(rng, 64, 8192)
        most = 8192 * 14336 * 4096
        k = max(64, min(k, most // (rows * n)))
        groups = 1 if rng.random() < 0.5 else _log(rng, 2, 32)
        while groups > 1 and groups * n * k > 2 ** 28:
            groups //= 2
        return {"op": op, "rows": rows, "n": n, "k": k, "groups": groups, "dtype": rng.choice(["bf16", "f16"])}
    experts = rng.choice([_log(rng, 4, 512), 8, 64, 256])
    return {"op": op, "rows": _log(rng, 1, 65536), "experts": experts, "k": rng.randint(1, min(experts, 8)),
            "dtype": dtype, "renormalize": rng.random() < 0.5}


# ------------------------------------------------------------------------------------ inputs

def _activations(gen, rows, cols, dtype):
    """Activations as a network has them: channels of uneven size, a few of them large, and
    some rows of zeros (padding)."""
    size = torch.exp(0.5 * torch.randn(cols, generator=gen, device="cuda"))
    size = torch.where(torch.rand(cols, generator=gen, device="cuda") < 0.004, size * 20, size)
    x = torch.randn(rows, cols, generator=gen, device="cuda") * size
    x *= (torch.rand(rows, 1, generator=gen, device="cuda") >= 0.03)
    return x.to(dtype)


def _gradient(gen, rows, cols, dtype):
    size = 0.05 * torch.exp(0.5 * torch.randn(rows, 1, generator=gen, device="cuda"))
    return (torch.randn(rows, cols, generator=gen, device="cuda") * size).to(dtype)


def _counts(seed, rows, groups):
    """Ragged group sizes that sum to rows; from four groups on one of them is empty."""
    rng = np.random.default_rng(seed)
    share = rng.dirichlet(np.full(groups, 4.0))
    if groups >= 4:
        share[int(rng.integers(groups))] = 0.0
        share /= share.sum()
    return [int(c) for c in rng.multinomial(rows, share)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype, rows = case["op"], _DTYPES[case["dtype"]], case["rows"]
    state = dict(case)
    if op == "checkpoint":
        state["x"] = _activations(gen, rows, case["cols"], dtype)
    elif op == "norm":
        cols = case["cols"]
        state["x"] = _activations(gen, rows, cols, dtype)
        state["w"] = (1 + 0.2 * torch.randn(cols, generator=gen, device="cuda")).to(_DTYPES[case["weight"]])
        state["dy"] = _gradient(gen, rows, cols, dtype)
    elif op == "swiglu":
        cols = case["cols"]
        if case["packed"]:
            state["gate_up"] = _activations(gen, rows, 2 * cols, dtype)
        else:
            state["gate"] = _activations(gen, rows, cols, dtype)
            state["up"] = _activations(gen, rows, cols, dtype)
        state["dh"] = _gradient(gen, rows, cols, dtype)
    elif op == "wgrad":
        state["x"] = _activations(gen, rows, case["k"], dtype)
        state["dy"] = _gradient(gen, rows, case["n"], dtype)
        if case["groups"] > 1:
            state["counts"] = _counts(seed, rows, case["groups"])
            state["offsets"] = torch.tensor([0, *np.cumsum(state["counts"]).tolist()], dtype=torch.int32,
                                            device="cuda")
    else:
        experts, k = case["experts"], case["k"]
        lean = 0.7 * torch.randn(experts, generator=gen, device="cuda")
        state["logits"] = (1.5 * torch.randn(rows, experts, generator=gen, device="cuda") + lean).to(dtype)
        state["valid"] = torch.rand(rows, generator=gen, device="cuda") >= 0.125
        state["dweights"] = torch.randn(rows, k, generator=gen, device="cuda") * 0.02
        state["dbalance"] = torch.full((), 0.01, device="cuda")
    return state


# --------------------------------------------------------------------------------- plain form

def _read_back(x):
    """The float32 values that the 8-bit checkpoint of x stands for."""
    low = -24 if x.dtype == torch.float16 else -126
    v = x.float()
    rows, cols = v.shape
    v = torch.nn.functional.pad(v, (0, -cols % _BLOCK)).view(rows, -1, _BLOCK)
    most = v.abs().amax(-1, keepdim=True)
    e = (torch.frexp(most).exponent - 7).clamp(min=low)
    v = torch.ldexp(torch.ldexp(v, -e).round().clamp(-127, 127), e)
    v = torch.where(torch.isfinite(most), v, torch.nan)
    return v.view(rows, -1)[:, :cols]


def _plain(state):
    op = state["op"]
    if op == "checkpoint":
        return {"values": _read_back(state["x"]).to(state["x"].dtype)}
    if op == "norm":
        x, w, dy = state["x"].float(), state["w"].float(), state["dy"].float()
        r = (x.square().mean(-1, keepdim=True) + _EPS).rsqrt()
        y = x * r * w
        v = _read_back(state["x"])
        g = w * dy
        dx = r * g - v * (r * r * r * (v * g).mean(-1, keepdim=True))
        return {"y": y.to(state["x"].dtype), "dx": dx.to(state["x"].dtype),
                "dw": (dy * v * r).sum(0).to(state["w"].dtype)}
    if op == "swiglu":
        gate, up = state["gate_up"].chunk(2, -1) if state["packed"] else (state["gate"], state["up"])
        g, u, dh = gate.float(), up.float(), state["dh"].float()
        h = g / (1 + torch.exp(-g)) * u
        g, u = _read_back(gate), _read_back(up)
        s = 1 / (1 + torch.exp(-g))
        dg = dh * u * s * (1 + g * (1 - s))
        du = dh * g * s
        out = {"h": h.to(gate.dtype)}
        if state["packed"]:
            return {**out, "dgate_up": torch.cat([dg, du], -1).to(gate.dtype)}
        return {**out, "dgate": dg.to(gate.dtype), "dup": du.to(gate.dtype)}
    if op == "wgrad":
        v, dy = _read_back(state["x"]), state["dy"].float()
        if state["groups"] == 1:
            return {"dw": (dy.t() @ v).to(state["dy"].dtype)}
        first, last = state["offsets"][:-1, None].long(), state["offsets"][1:, None].long()
        at = first + torch.arange(max(state["counts"]), device=v.device)
        inside = (at < last)[..., None]
        at = at.clamp(max=state["rows"] - 1)
        return {"dw": torch.bmm((dy[at] * inside).transpose(1, 2), v[at] * inside).to(state["dy"].dtype)}
    logits, valid, k = state["logits"].float(), state["valid"], state["k"]
    rows, experts = logits.shape
    n = valid.sum().clamp(min=1).float()
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    chosen = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :k]
    weights = p.gather(1, chosen)
    total = weights.sum(-1, keepdim=True) if state["renormalize"] else torch.ones_like(weights[:, :1])
    weights = weights / total * valid[:, None]
    hit = torch.zeros(rows, experts, dtype=torch.int32, device=p.device)
    hit.scatter_(1, chosen, valid[:, None].to(torch.int32).expand(rows, k))
    counts = hit.sum(0, dtype=torch.int32)
    share = counts.float() * (experts / (k * n))
    balance = (share * ((p * valid[:, None]).sum(0) / n)).sum()
    dw = state["dweights"] * valid[:, None]
    if state["renormalize"]:
        dw = (dw - (dw * weights).sum(-1, keepdim=True)) / total
    g = (share * (state["dbalance"] / n)).expand(rows, experts).scatter_add(1, chosen, dw)
    dlogits = p * (g - (p * g).sum(-1, keepdim=True)) * valid[:, None]
    return {"weights": weights, "experts": torch.where(valid[:, None], chosen, -1).to(torch.int32),
            "counts": counts, "balance": balance, "dlogits": dlogits.to(state["logits"].dtype)}


# ---------------------------------------------------------------------- the framework's calls

def _own(state):
    from adamw4bit_b200 import activations as A
    from adamw4bit_b200 import routing as R

    op = state["op"]
    if op == "checkpoint":
        return {"values": A.dequantize_act8(A.quantize_act8(state["x"]))}
    if op == "norm":
        y, saved = A.rms_norm_forward(state["x"], state["w"], eps=_EPS)
        dx, dw = A.rms_norm_backward(state["dy"], state["w"], saved)
        return {"y": y, "dx": dx, "dw": dw}
    if op == "swiglu":
        if state["packed"]:
            h, saved = A.swiglu_forward(state["gate_up"])
            return {"h": h, "dgate_up": A.swiglu_backward(state["dh"], saved)}
        h, saved = A.swiglu_forward(state["gate"], state["up"])
        dgate, dup = A.swiglu_backward(state["dh"], saved)
        return {"h": h, "dgate": dgate, "dup": dup}
    if op == "wgrad":
        x8 = A.quantize_act8(state["x"])
        return {"dw": A.weight_grad(state["dy"], x8, offsets=state.get("offsets"))}
    routed = R.route_forward(state["logits"], state["k"], valid=state["valid"], renormalize=state["renormalize"])
    dlogits = R.route_backward(state["dweights"], state["dbalance"], routed)
    return {"weights": routed.weights, "experts": routed.experts, "counts": routed.counts,
            "balance": routed.balance_loss, "dlogits": dlogits}


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------------------- work

def _held(rows, cols):
    """Bytes of a checkpoint: a byte for each value and one for each block."""
    return rows * (cols + -(-cols // _BLOCK))


def work(case):
    """Bytes that each call has to read and write once, and operations.  The checkpoint is
    written by a forward call and read by a backward call, and counts in both."""
    op, rows, size = case["op"], case["rows"], _BYTES[case["dtype"]]
    if op == "checkpoint":
        cols = case["cols"]
        return {"bytes": 2 * rows * cols * size + 2 * _held(rows, cols), "flops": 4 * rows * cols}
    if op == "norm":
        cols = case["cols"]
        # forward reads x, w and writes y, checkpoint, r; backward reads dy, w, checkpoint, r and writes dx, dw
        return {"bytes": 4 * rows * cols * size + 2 * _held(rows, cols) + 8 * rows + 3 * cols * _BYTES[case["weight"]],
                "flops": 18 * rows * cols}
    if op == "swiglu":
        cols = case["cols"]
        # forward reads g, u and writes h, two checkpoints; backward reads dh, both and writes dg, du
        return {"bytes": 6 * rows * cols * size + 4 * _held(rows, cols), "flops": 30 * rows * cols}
    if op == "wgrad":
        n, k, groups = case["n"], case["k"], case["groups"]
        return {"bytes": rows * (n + k) * size + 2 * _held(rows, k) + groups * n * k * size,
                "flops": 2 * rows * n * k + 2 * rows * k}
    experts, k = case["experts"], case["k"]
    # forward reads logits and mask, writes weights, indices and counts; backward reads logits,
    # mask, indices, weights, their gradient and counts, and writes dlogits
    return {"bytes": 3 * rows * experts * size + rows * (2 + 20 * k) + 8 * experts,
            "flops": 20 * rows * experts}


# ----------------------------------------------------------------------------- 64-bit values

def _exact_values(x):
    """The checkpoint's values in float64, the exponent taken from the bits of the block's
    largest magnitude."""
    low = -24 if x.dtype == torch.float16 else -126
    rows, cols = x.shape
    blocks = -(-cols // _BLOCK)
    v = torch.zeros(rows, blocks * _BLOCK, dtype=torch.float64, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, blocks, _BLOCK)
    most = v.abs().amax(-1, keepdim=True)
    e = ((most.view(torch.int64) >> 52) - 1023 - 6).clamp(min=low)
    unit = ((e + 1023) << 52).view(torch.float64)
    q = torch.round(v / unit)
    q = torch.minimum(torch.maximum(q, torch.full_like(q, -127)), torch.full_like(q, 127))
    v = torch.where(torch.isfinite(most), q * unit, torch.full_like(q, math.nan))
    return v.reshape(rows, blocks * _BLOCK)[:, :cols]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "checkpoint":
        return {"values": _exact_values(state["x"])}
    if op == "norm":
        x, w, dy = (state[name].double() for name in ("x", "w", "dy"))
        r = 1 / torch.sqrt((x * x).sum(-1) / case["cols"] + _EPS)
        y = torch.einsum("tc,t,c->tc", x, r, w)
        v = _exact_values(state["x"])
        inner = torch.einsum("tc,tc,c->t", v, dy, w) / case["cols"]
        dx = r[:, None] * dy * w - v * (r ** 3 * inner)[:, None]
        return {"y": y, "dx": dx, "dw": torch.einsum("tc,tc,t->c", dy, v, r)}
    if op == "swiglu":
        cols = case["cols"]
        if case["packed"]:
            gate, up = state["gate_up"][:, :cols], state["gate_up"][:, cols:]
        else:
            gate, up = state["gate"], state["up"]
        h = gate.double() * torch.sigmoid(gate.double()) * up.double()
        g, u, dh = _exact_values(gate), _exact_values(up), state["dh"].double()
        s = torch.sigmoid(g)
        dg = (s + g * s * (1 - s)) * u * dh
        du = s * g * dh
        if case["packed"]:
            return {"h": h, "dgate_up": torch.cat([dg, du], -1)}
        return {"h": h, "dgate": dg, "dup": du}
    if op == "wgrad":
        v, dy = _exact_values(state["x"]), state["dy"].double()
        if case["groups"] == 1:
            return {"dw": torch.einsum("tn,tk->nk", dy, v)}
        parts = [d.t() @ x for d, x in zip(dy.split(state["counts"]), v.split(state["counts"]))]
        return {"dw": torch.stack(parts)}
    logits, valid, k = state["logits"].double(), state["valid"], case["k"]
    rows, experts = logits.shape
    n = max(1, int(valid.sum()))
    p = torch.softmax(logits, -1)
    # descending by logit, then ascending by index
    order = np.argsort(-logits.cpu().numpy(), axis=-1, kind="stable")[:, :k]
    chosen = torch.from_numpy(np.ascontiguousarray(order)).to(logits.device)
    picked = torch.nn.functional.one_hot(chosen, experts).to(torch.float64)
    picked[~valid] = 0
    counts = picked.sum((0, 1))
    mean = p[valid].sum(0) / n
    share = experts * counts / (k * n)
    total = p.gather(1, chosen).sum(-1, keepdim=True) if case["renormalize"] else torch.ones_like(p[:, :1])
    weights = p.gather(1, chosen) / total
    # d weights_j / d l_i = weights_j (delta_ij - q_i), q the softmax over the chosen or over all
    scaled = state["dweights"].double() * weights
    base = picked.mul(weights[..., None]).sum(1) if case["renormalize"] else p
    dlogits = picked.mul(scaled[..., None]).sum(1) - base * scaled.sum(-1, keepdim=True)
    dlogits = dlogits + state["dbalance"].double() / n * p * (share - (p @ share)[:, None])
    dlogits[~valid] = 0
    weights[~valid] = 0
    return {"weights": weights, "experts": torch.where(valid[:, None], chosen, -1).to(torch.int32),
            "counts": counts.to(torch.int32), "balance": (share * mean).sum(), "dlogits": dlogits}
