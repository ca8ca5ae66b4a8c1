"""RMS norm of very large and very small rows: its gradient as long as the sum of squares is a normal float32."""

from __future__ import annotations

import pytest
import torch

from adamw4bit_b200 import activations as A
from tests.test_gpu_activations import DEV, _check_norm, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [-58, -45, -41, 41, 45, 55])
@pytest.mark.parametrize("shape", [(9, 24), (7, 1000), (5, 4096), (3, 8191)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
def test_gradient_of_rows_of_any_size(dtype, shape, power):
    x = (_randn(*shape).clamp(-16, 16) * 2.0 ** power).to(dtype)
    dy = _randn(*shape, seed=1, dtype=dtype, scale=0.1)
    w = (1 + 0.3 * _randn(shape[-1], seed=2)).to(dtype)
    y, saved = A.rms_norm_forward(x.to(DEV), w.to(DEV), 0.0)
    dx, dw = A.rms_norm_backward(dy.to(DEV), w.to(DEV), saved)
    assert dx.isfinite().all() and dw.isfinite().all()
    _check_norm(x, w, dy, y, saved, dx, dw, 0.0)
