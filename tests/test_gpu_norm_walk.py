"""RMS norm over more rows than are resident, for every number of threads a row, against float64 on the device.

Blocks stay and walk the rows; here every thread has two rows or more, and the last round is not full.
A sum's error is bounded by the additions that a term goes through, not by their number:

    mean(x^2), the dot product    16 values a thread, 5 shuffles, up to 32 warps: 46 additions; r has half of it
    dw                            a thread's rows, 5 shuffles, 4 warps, a 32nd of the blocks, 5 shuffles: under 64
"""

from __future__ import annotations

import pytest
import torch

from adamw4bit_b200 import activations as A
from tests import act8_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
EPS32 = 2.0 ** -24
# the widest row of each number of threads, and rows off 16 bytes
WHOLE = {64: 8, 128: 16, 256: 32, 512: 32, 1024: 64, 1536: 96, 2048: 128, 2560: 160, 4096: 256, 5120: 320, 6144: 384,
         7168: 448, 8192: 512, 12288: 768, 16384: 1024}
ODD = {61: 8, 125: 16, 255: 32, 511: 32, 1021: 64, 2047: 128, 4093: 256, 8191: 512, 16381: 1024}


def _within(got, ref, dtype, slack):
    off = (got.double() - ref).abs() - (1.02 * R.UNIT[dtype] * ref.abs() + R.STEP[dtype] + slack)
    assert off.max() <= 0, f"off by {off.max().item():.3g} more than allowed"


@pytest.mark.parametrize("cols,threads", [*WHOLE.items(), *ODD.items()])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["float32", "bfloat16", "float16"])
def test_every_row_of_a_walk(dtype, cols, threads):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    resident = sms * max(1, 1024 // threads)
    rows = resident * 5 // 2 + 13
    g = torch.Generator(DEV).manual_seed(cols)
    size = torch.exp(torch.randn(rows, 1, generator=g, device=DEV))       # rows differ, so that one in another's place shows
    x = (torch.randn(rows, cols, generator=g, device=DEV) * size).to(dtype)
    dy = (0.1 * torch.randn(rows, cols, generator=g, device=DEV)).to(dtype)
    w = 1 + 0.3 * torch.randn(cols, generator=g, device=DEV)
    y, saved = A.rms_norm_forward(x, w, 1e-5, checkpoint_output=True)
    dx, dw = A.rms_norm_backward(dy, w, saved)
    of_x, of_y = A.quantize_act8(x), A.quantize_act8(y)
    for mine, ref in ((saved.x8, of_x), (saved.output, of_y)):
        assert torch.equal(mine.codes, ref.codes) and torch.equal(mine.scales, ref.scales)
    ref, r = R.rms_norm(x, w, 1e-5)
    few = 32 * EPS32
    _within(saved.rstd[:, None], r, torch.float32, few * r)
    _within(y, ref, dtype, few * ref.abs())
    gx, mx, gw, mw = R.rms_norm_backward(dy, w, of_x.dequantize().double(), r)
    _within(dx, gx, dtype, (4 * few + 64 * EPS32) * mx)
    _within(dw, gw, torch.float32, (few + 64 * EPS32) * mw)


@pytest.mark.parametrize("cols", [40, 96, 1000, 4096, 4099])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["float32", "bfloat16", "float16"])
def test_a_row_of_zeros_without_eps(dtype, cols):
    x = torch.randn(5, cols, generator=torch.Generator(DEV).manual_seed(1), device=DEV).to(dtype)
    x[2] = 0
    w = torch.ones(cols, device=DEV)
    y, saved = A.rms_norm_forward(x, w, 0.0)
    assert saved.rstd[2].isposinf() and saved.rstd[[0, 1, 3, 4]].isfinite().all()
    assert y[2].isnan().all() and y[[0, 1, 3, 4]].isfinite().all()        # 0 times infinity, as in the formula
    ref, _ = R.rms_norm(x[[0, 1, 3, 4]], w, 0.0)
    _within(y[[0, 1, 3, 4]], ref, dtype, 32 * EPS32 * ref.abs())


def test_weight_grad_added_to_float16():
    g = torch.Generator(DEV).manual_seed(2)
    x = torch.randn(300, 264, generator=g, device=DEV).half()
    dy = (0.1 * torch.randn(300, 130, generator=g, device=DEV)).half()
    start = torch.randn(130, 264, generator=g, device=DEV).half()
    x8, total = A.quantize_act8(x), start.clone()
    assert A.weight_grad(dy, x8, out=total, accumulate=True) is total
    v = x8.dequantize().double()
    ref, mag = dy.double().t() @ v + start.double(), dy.double().abs().t() @ v.abs() + start.double().abs()
    _within(total, ref, torch.float16, 2 * 302 * EPS32 * mag)
