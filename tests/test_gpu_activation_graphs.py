"""The activation and router calls in a CUDA graph: replayed on other inputs they give what plain calls give."""

from __future__ import annotations

import pytest
import torch

from adamw4bit_b200 import activations as A
from adamw4bit_b200 import routing as Q

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _randn(*shape, seed, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator(DEV).manual_seed(seed), device=DEV).to(dtype)


def _norm(x, dy):
    w = torch.ones(256, device=DEV, dtype=x.dtype)
    y, saved = A.rms_norm_forward(x, w, checkpoint_output=True)
    return (y, saved.output.dequantize(), *A.rms_norm_backward(dy, w, saved))


def _glu(x, dy):
    h, saved = A.swiglu_forward(x, dy, checkpoint_output=True)
    return (h, saved.output.dequantize(), *A.swiglu_backward(dy, saved))


def _route(x, dy):
    r = Q.route_forward(x, 4)
    return r.weights, r.experts, r.counts, r.balance_loss, Q.route_backward(dy[:, :4].float(), torch.ones((), device=DEV), r)


def _groups(x, dy):
    offsets = Q.group_offsets(Q.route_forward(x[:, :5], 1).counts)
    return A.weight_grad(dy, A.quantize_act8(x), offsets),


def _autograd(x, dy):
    w = torch.ones(64, 256, device=DEV, dtype=x.dtype, requires_grad=True)
    x = x.detach().requires_grad_()
    return torch.autograd.grad(A.linear(A.swiglu(x, x), w), (x, w), dy[:, :64])


@pytest.mark.parametrize("calls", [_norm, _glu, _route, _groups, _autograd], ids=lambda f: f.__name__[1:])
def test_replayed_on_other_inputs(calls):
    x, dy = _randn(5000, 256, seed=1), _randn(5000, 256, seed=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls(x, dy)                                      # the warm-up call
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls(x, dy)
    for seed in (3, 5):
        x.copy_(_randn(5000, 256, seed=seed))
        dy.copy_(_randn(5000, 256, seed=seed + 1))
        graph.replay()
        for got, want in zip(out, calls(x, dy)):
            assert torch.equal(got, want)


def test_grouped_linear_refuses_a_capture():
    x, w = _randn(10, 64, seed=1), _randn(2, 8, 64, seed=2)
    offsets = torch.tensor([0, 4, 10], dtype=torch.int32, device=DEV)
    want = A.grouped_linear(x, w, offsets)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            A.grouped_linear(x, w, offsets)
        y = x + 1
    graph.replay()
    assert torch.equal(y, x + 1) and torch.equal(A.grouped_linear(x, w, offsets), want)
