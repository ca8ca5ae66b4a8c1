"""A weight gradient whose kernel gives up its waits: NaN in the result, an error on the host, and the next call works.

The limit of 0 gives every wait up at once, before a copy or a product is issued."""

from __future__ import annotations

import pytest
import torch

from adamw4bit_b200 import ZEEDENAdamW4Bit
from adamw4bit_b200 import _native as N
from adamw4bit_b200 import activations as A

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture
def no_waits():
    A.check_weight_grads(0)
    N.check(N.lib().aw4_set_wait_limit(0), "aw4_set_wait_limit")
    try:
        yield
    finally:
        N.check(N.lib().aw4_set_wait_limit(2 ** 63), "aw4_set_wait_limit")
        torch.cuda.synchronize()
        N._wait_words[0].zero_()


def _inputs(rows, n, k, dtype=torch.bfloat16):
    g = torch.Generator(DEV).manual_seed(rows)
    x = torch.randn(rows, k, generator=g, device=DEV).to(dtype)
    return torch.randn(rows, n, generator=g, device=DEV).to(dtype), A.quantize_act8(x)


@pytest.mark.parametrize("rows,n,k,counts,dtype,out", [
    (64, 40, 33, None, torch.bfloat16, None),
    (300, 600, 411, None, torch.float16, torch.float32),
    (8192, 600, 300, None, torch.bfloat16, None),                       # cut tiles
    (4110, 600, 300, [4000, 10, 0, 100], torch.bfloat16, torch.float32),
    (700, 136, 300, [100, 0, 600], torch.float16, None),
], ids=str)
def test_nothing_stands_as_a_number(no_waits, rows, n, k, counts, dtype, out):
    dy, x8 = _inputs(rows, n, k, dtype)
    offsets = None
    if counts:
        offsets = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    shape = (n, k) if offsets is None else (len(counts), n, k)
    dw = A.weight_grad(dy, x8, offsets, out=torch.zeros(shape, dtype=out or dtype, device=DEV))
    with pytest.raises(N.NativeError, match="not complete"):
        A.check_weight_grads(DEV)
    assert dw.isnan().all()
    total = torch.ones(shape, dtype=out or dtype, device=DEV)
    A.weight_grad(dy, x8, offsets, out=total, accumulate=True)
    torch.cuda.synchronize()
    with pytest.raises(N.NativeError, match="not complete"):
        A.weight_grad(dy, x8, offsets)                                  # the next call on the device says it too
    assert total.isnan().all()


def test_the_next_call_works(no_waits):
    dy, x8 = _inputs(200, 64, 96)
    A.weight_grad(dy, x8)
    N.check(N.lib().aw4_set_wait_limit(2 ** 63), "aw4_set_wait_limit")
    with pytest.raises(N.NativeError):
        A.check_weight_grads()
    dw = A.weight_grad(dy, x8, out_dtype=torch.float32)
    A.check_weight_grads()
    ref = dy.double().t() @ x8.dequantize().double()
    mag = dy.double().abs().t() @ x8.dequantize().double().abs()
    assert ((dw.double() - ref).abs() <= 2 * 202 * 2.0 ** -24 * mag).all()


def test_a_replayed_graph_and_the_optimizer(no_waits):
    x = torch.randn(128, 64, device=DEV, dtype=torch.bfloat16)
    w = torch.nn.Parameter(torch.randn(48, 64, device=DEV, dtype=torch.bfloat16))
    opt = ZEEDENAdamW4Bit([w])
    dy = torch.randn(128, 48, device=DEV, dtype=torch.bfloat16)
    x8 = A.quantize_act8(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dw = A.weight_grad(dy, x8)
    dw.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert dw.isnan().all()
    before = w.detach().clone()
    w.grad = dw
    with pytest.raises(N.NativeError, match="not complete"):
        opt.step()
    assert torch.equal(before, w.detach())
