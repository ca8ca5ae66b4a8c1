"""What the activation and router entry points refuse, and the checkpoint's definition.  No GPU: a bad
argument is answered before a device is looked at."""

from __future__ import annotations

import math

import pytest
import torch

import adamw4bit_b200
from adamw4bit_b200 import _native as N
from adamw4bit_b200 import activations as A
from adamw4bit_b200 import routing as Q
from tests import act8_reference as R

P = 4096            # an address that is never followed
INVALID, UNSUPPORTED, OK = N.AW4_ERR_INVALID, N.AW4_ERR_UNSUPPORTED, N.AW4_OK


def _call(name, *args):
    return getattr(N.lib(), name)(*args, 0, None)


def test_modules_are_public():
    assert adamw4bit_b200.activations is A and adamw4bit_b200.routing is Q


def test_nothing_to_do_is_fine():
    assert _call("aw4_act8_quantize", None, N.F32, 0, 64, 64, None, None) == OK
    assert _call("aw4_act8_dequantize", None, None, N.BF16, 4, 0, None, 0) == OK
    assert _call("aw4_swiglu_forward", None, None, N.F16, 0, 8, 8, 8, *[None] * 7) == OK
    assert _call("aw4_weight_grad", None, N.BF16, 8, 0, 0, None, None, 4, None, 1, None, N.BF16, 0, None, 0, None) == OK


@pytest.mark.parametrize("name,args,code", [
    ("aw4_act8_quantize", (P, 7, 1, 32, 32, P, P), INVALID),
    ("aw4_act8_quantize", (P, N.F32, -1, 32, 32, P, P), INVALID),
    ("aw4_act8_quantize", (P, N.F32, 1, 1 << 31, 1 << 31, P, P), UNSUPPORTED),
    ("aw4_act8_quantize", (P, N.F32, 1 << 50, 1 << 20, 32, P, P), UNSUPPORTED),
    ("aw4_act8_quantize", (None, N.F32, 1, 32, 32, P, P), INVALID),
    ("aw4_act8_quantize", (P, N.F32, 1, 32, 32, P + 8, P), INVALID),
    ("aw4_act8_dequantize", (P, None, N.F32, 1, 32, P, 32), INVALID),
    ("aw4_rms_norm_forward", (P, N.F32, 1, 16385, 16385, P, N.F32, 0.0, P, P, P, P, None, None), UNSUPPORTED),
    ("aw4_rms_norm_forward", (P, N.F32, 1, 32, 32, P, 5, 0.0, P, P, P, P, None, None), INVALID),
    ("aw4_rms_norm_forward", (P, N.F32, 1, 32, 32, P, N.F32, 0.0, P, P, P, P, P, None), INVALID),
    ("aw4_rms_norm_backward", (P, N.F32, 1, 16385, 16385, P, P, P, P, N.F32, P, P, P, 0), UNSUPPORTED),
    ("aw4_rms_norm_backward", (P, N.F32, 1, 32, 32, P, P, P, P, N.F32, P, None, P, 0), INVALID),
    ("aw4_swiglu_forward", (P, P, N.F32, 1, 32, 32, 32, P, P, P, P, P, P, None), INVALID),
    ("aw4_swiglu_forward", (P, None, N.F32, 1, 32, 32, 32, P, P, P, P, P, None, None), INVALID),
    ("aw4_swiglu_backward", (P, N.F32, 1, 32, 32, P + 4, P, P, P, P, P, 32), INVALID),
    ("aw4_weight_grad", (P, N.F32, 8, 8, 8, P, P, 8, None, 1, P, N.F32, 0, P, 0, None), UNSUPPORTED),
    ("aw4_weight_grad", (P, N.BF16, 8, 8, 8, P, P, 8, None, 1, P, N.F16, 0, P, 0, None), UNSUPPORTED),
    ("aw4_weight_grad", (P, N.BF16, 8, 8, 8, P, P, 8, None, 2, P, N.BF16, 0, P, 0, None), INVALID),
    ("aw4_weight_grad", (P, N.BF16, -8, 8, 8, P, P, 8, None, 1, P, N.BF16, 0, P, 0, None), INVALID),
    ("aw4_weight_grad", (P, N.BF16, 8, 8, 8, P, P, 8, P, 70000, P, N.BF16, 0, P, 0, None), UNSUPPORTED),
    ("aw4_weight_grad", (P, N.BF16, 8, 8, 8, P, P, 8, None, 1, P + 1, N.BF16, 0, P, 0, None), INVALID),
    ("aw4_route_forward", (P, N.F32, 4, 8, 8, 9, None, 1, *[P] * 7, 0), INVALID),
    ("aw4_route_forward", (P, N.F32, 4, 8, 8, 0, None, 1, *[P] * 7, 0), INVALID),
    ("aw4_route_forward", (P, N.F32, 4, 1025, 1025, 2, None, 1, *[P] * 7, 0), UNSUPPORTED),
    ("aw4_route_forward", (P, N.F32, 1 << 31, 8, 8, 2, None, 1, *[P] * 7, 0), UNSUPPORTED),
    ("aw4_route_forward", (P, 3, 4, 8, 8, 2, None, 1, *[P] * 7, 0), INVALID),
    ("aw4_route_backward", (P, N.F32, 4, 8, 8, 2, 1, P, P, P + 4, P, P, P, P, P), INVALID),
    ("aw4_route_backward", (P, N.F32, 4, 8, 8, 2, 1, None, P, P, P, P, P, P, P), INVALID),
])
def test_bad_arguments_are_answered_on_the_host(name, args, code):
    assert _call(name, *args) == code
    assert name[4:].split("_")[0] in N.lib().aw4_last_error().decode()


def test_python_entry_points_want_cuda_tensors():
    x = torch.ones(4, 64)
    for call in (lambda: A.quantize_act8(x), lambda: A.rms_norm(x, x[0]), lambda: A.swiglu(x),
                 lambda: A.linear(x.half(), x.half()), lambda: Q.route(x, 2)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        A.linear(x, x)
    with pytest.raises(ValueError):
        Q.group_offsets(x)
    assert Q.group_offsets(torch.tensor([2, 0, 3], dtype=torch.int32)).tolist() == [0, 2, 2, 5]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_the_definition(dtype):
    """A value is off by at most half a step, 1/128 of its block's largest magnitude, and by a step only where
    it would round to 128 steps; what reads back encodes to itself; it is exact in the dtype."""
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(50, 200, generator=g) * torch.exp(2 * torch.randn(200, generator=g))).to(dtype)
    codes, scales = R.encode(x)
    assert codes.shape == (50, 224) and scales.shape == (50, 7) and codes.abs().max() <= 127
    assert not codes[:, 200:].any()
    back = R.decode(codes, scales, 200)
    step = torch.ldexp(torch.ones(scales.shape, dtype=torch.float64), scales - 127).repeat_interleave(32, 1)[:, :200]
    off = (back - x.double()).abs() / step
    assert off.max() <= 1 and (off[x.double().abs() < 127.5 * step] <= 0.5).all()
    assert torch.equal(back.to(dtype).double(), back)
    again, exponents = R.encode(back.to(dtype))
    assert torch.equal(R.decode(again, exponents, 200), back)


def test_the_definition_at_the_edges():
    x = torch.tensor([[math.inf] + [1.0] * 31 + [0.0] * 32 + [torch.finfo(torch.float32).max] * 32 + [2.0 ** -140] * 4])
    codes, scales = R.encode(x)
    assert scales.tolist() == [[255, 1, 127 + 121, 1]]
    back = R.decode(codes, scales, 100)
    assert torch.isnan(back[0, :32]).all() and not back[0, 32:64].any() and torch.isfinite(back[0, 64:96]).all()
    assert back[0, 64] == 127 * 2.0 ** 121 and not back[0, 96:].any()
    assert R.encode(torch.full((1, 1), 2.0 ** -24).half())[0][0, 0] == 1
