"""8-bit activation checkpoints, and the backward passes that read them.

A training step holds its optimizer moments in 4 bits; this module holds the other large buffer, the
activations that wait for the backward pass, in 8.  Values are cut into blocks of 32 along the last
axis; a block keeps 32 signed bytes q and one exponent byte and stands for q * 2^e (1.03 bytes a value):

    e = max(floor(log2(max |x|)) - 6, e_min)     e_min = -24 for float16, else -126
    q = clamp(round_half_even(x * 2^-e), -127, 127)

A block with an infinity or a NaN reads back as NaN.  Every value q * 2^e is exact in bfloat16 and
float16, so the tensor cores multiply checkpoints without another rounding.

=====================  ==================================================================
``quantize_act8``      a tensor's checkpoint (:class:`Act8`); ``dequantize_act8`` reads it back
``rms_norm``           y = x (mean(x^2) + eps)^-1/2 w, keeps the checkpoint of x
``swiglu``             h = gate sigmoid(gate) up, keeps the checkpoints of gate and up
``linear``             x W^T + b, keeps the checkpoint of x for ``weight_grad``
``grouped_linear``     the same over groups of rows, one weight each (experts)
=====================  ==================================================================

The functions of the table are differentiable.  ``*_forward`` / ``*_backward`` and ``weight_grad`` are
the calls below them, for code that runs its own backward pass.  Everything runs on the current
stream of the tensors' device; a tensor or checkpoint that belongs to another stream is the caller's
to order (``Act8.record_stream``).  There is no CPU path.
"""

from __future__ import annotations

import functools
import math
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as N

__all__ = [
    "Act8", "RMSNormSaved", "SwiGLUSaved", "quantize_act8", "dequantize_act8", "rms_norm",
    "rms_norm_forward", "rms_norm_backward", "swiglu", "swiglu_forward", "swiglu_backward", "linear",
    "grouped_linear", "weight_grad", "check_weight_grads",
]

BLOCK = 32


class Act8:
    """The 8-bit checkpoint of a tensor: its codes and block exponents in a buffer (``data``, from byte
    ``start`` on), and the shape and dtype it reads back as.  ``codes`` is int8 [rows, cols rounded up to 32], ``scales`` uint8
    [rows, blocks] with e + 127 (255: the block was not finite)."""

    __slots__ = ("data", "shape", "dtype", "rows", "cols", "start")

    def __init__(self, data: torch.Tensor, shape, dtype: torch.dtype, start: int = 0):
        self.data, self.shape, self.dtype, self.start = data, shape, dtype, start
        self.cols = shape[-1]
        self.rows = math.prod(shape[:-1])

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def nbytes(self) -> int:
        return self.rows * -(-self.cols // BLOCK) * (BLOCK + 1)

    @property
    def codes(self) -> torch.Tensor:
        pitch = -(-self.cols // BLOCK) * BLOCK
        return self.data[self.start: self.start + self.rows * pitch].view(torch.int8).view(self.rows, pitch)

    @property
    def scales(self) -> torch.Tensor:
        blocks = -(-self.cols // BLOCK)
        return self.data[self.start + self.rows * blocks * BLOCK: self.start + self.nbytes].view(self.rows, blocks)

    def dequantize(self) -> torch.Tensor:
        return dequantize_act8(self)

    def record_stream(self, stream) -> None:
        self.data.record_stream(stream)

    def __repr__(self) -> str:
        return f"Act8(shape={tuple(self.shape)}, dtype={self.dtype}, device={self.device})"


def _empty_act8(t: torch.Tensor, shape, rows: int, cols: int, more: int = 0) -> Act8:
    """A checkpoint to be written for a tensor like t of this shape, and `more` bytes behind it."""
    x8 = Act8.__new__(Act8)
    x8.data = t.new_empty(rows * (-(-cols // BLOCK)) * (BLOCK + 1) + more, dtype=torch.uint8)
    x8.shape, x8.dtype, x8.rows, x8.cols, x8.start = shape, t.dtype, rows, cols, 0
    return x8


def _second_act8(x8: Act8, start: int) -> Act8:
    """Another checkpoint like x8 in the same buffer."""
    y8 = Act8.__new__(Act8)
    y8.data, y8.shape, y8.dtype, y8.rows, y8.cols, y8.start = x8.data, x8.shape, x8.dtype, x8.rows, x8.cols, start
    return y8


def _ptrs(x8: Act8) -> tuple[int, int]:
    """Addresses of codes and scales."""
    p = x8.data.data_ptr() + x8.start
    return p, p + x8.rows * (-(-x8.cols // BLOCK)) * BLOCK


def _second_start(rows: int, cols: int) -> int:
    """Where a second checkpoint, or float32 statistics, begin behind a first: on 16 bytes."""
    return -(-(rows * (-(-cols // BLOCK)) * (BLOCK + 1)) // 16) * 16


class RMSNormSaved(NamedTuple):
    """What ``rms_norm_forward`` keeps: the checkpoint of x, and behind it in the same buffer
    (mean(x^2) + eps)^-1/2 of its rows.  ``output`` is the checkpoint of y where it was asked for."""
    x8: Act8
    output: Act8 | None = None

    @property
    def rstd(self) -> torch.Tensor:
        start = _second_start(self.x8.rows, self.x8.cols)
        return self.x8.data[start: start + 4 * self.x8.rows].view(torch.float32)


class SwiGLUSaved(NamedTuple):
    """What ``swiglu_forward`` keeps: the checkpoints of gate and up; ``packed`` where they came as halves
    of one tensor.  ``output`` is the checkpoint of h where it was asked for."""
    gate8: Act8
    up8: Act8
    packed: bool
    output: Act8 | None = None


def _dtype_code(t: torch.Tensor, what: str) -> int:
    code = N.DTYPE_CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: float32, bfloat16 or float16 expected, found {t.dtype}")
    return code


def _rows_of(t: torch.Tensor, what: str) -> tuple[torch.Tensor, int, int, int]:
    """t as rows of its last axis: (tensor, rows, cols, row stride).  A tensor whose leading axes have no
    single stride, or whose last axis is not contiguous, is copied."""
    if not t.is_cuda:
        N.require_cuda(t, what)
    shape = t.shape
    if not shape:
        raise ValueError(f"{what}: a tensor of at least one dimension expected")
    cols = shape[-1]
    rows = shape[0] if len(shape) == 2 else math.prod(shape[:-1])
    if t.is_contiguous():
        return t, rows, cols, cols
    if cols <= 1 or t.stride(-1) == 1:
        ld, size = None, 1
        for d in range(len(shape) - 2, -1, -1):
            if shape[d] == 1:
                continue
            if ld is None:
                ld, size = t.stride(d), shape[d]
            elif t.stride(d) == ld * size:
                size *= shape[d]
            else:
                break
        else:
            return t, rows, cols, cols if ld is None else ld
    return t.contiguous(), rows, cols, cols


def _same(a: torch.Tensor, device: torch.device, dtype: torch.dtype | None, what: str) -> None:
    if a.device != device:
        N.require_cuda(a, what)
        raise ValueError(f"{what}: on {a.device}, the others on {device}")
    if dtype is not None and a.dtype != dtype:
        raise TypeError(f"{what}: {dtype} expected, found {a.dtype}")


# ---------------------------------------------------------------------------
# checkpoint
# ---------------------------------------------------------------------------

def quantize_act8(x: torch.Tensor) -> Act8:
    """The 8-bit checkpoint of x, blocks of 32 along its last axis."""
    code = _dtype_code(x, "quantize_act8")
    src, rows, cols, ld = _rows_of(x, "quantize_act8")
    out = _empty_act8(x, x.shape, rows, cols)
    codes, scales = _ptrs(out)
    dev = x.get_device()
    N.check(N.lib().aw4_act8_quantize(src.data_ptr(), code, rows, cols, ld, codes, scales, dev,
                                      N.stream_of(dev)), "aw4_act8_quantize")
    return out


def dequantize_act8(x8: Act8) -> torch.Tensor:
    """The values a checkpoint stands for, in its shape and dtype."""
    out = x8.data.new_empty(x8.shape, dtype=x8.dtype)
    codes, scales = _ptrs(x8)
    dev = out.get_device()
    N.check(N.lib().aw4_act8_dequantize(codes, scales, N.DTYPE_CODES[x8.dtype], x8.rows, x8.cols,
                                        out.data_ptr(), x8.cols, dev, N.stream_of(dev)), "aw4_act8_dequantize")
    return out


# ---------------------------------------------------------------------------
# RMS norm
# ---------------------------------------------------------------------------

@functools.lru_cache(maxsize=1024)
def _norm_workspace(rows: int, cols: int, device: int) -> int:
    return int(N.lib().aw4_rms_norm_backward_workspace(rows, cols, device))


def _check_weight(weight: torch.Tensor, cols: int, x_dtype: torch.dtype, device, what: str) -> torch.Tensor:
    _same(weight, device, None, f"{what}: weight")
    if weight.shape != (cols,):
        raise ValueError(f"{what}: weight of shape ({cols},) expected, found {tuple(weight.shape)}")
    if weight.dtype not in (x_dtype, torch.float32):
        raise TypeError(f"{what}: weight in {x_dtype} or float32 expected, found {weight.dtype}")
    return weight.contiguous()


def rms_norm_forward(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *,
                     checkpoint_output: bool = False) -> tuple[torch.Tensor, RMSNormSaved]:
    """y = x r w with r = (mean(x^2) + eps)^-1/2 over the last axis (at most 16384 values), and what the
    backward call needs.  ``checkpoint_output`` also gives the checkpoint of y (``saved.output``), for a
    ``linear`` that reads y."""
    code = _dtype_code(x, "rms_norm")
    src, rows, cols, ld = _rows_of(x, "rms_norm")
    weight = _check_weight(weight, cols, x.dtype, x.device, "rms_norm")
    dev = x.get_device()
    y = x.new_empty(x.shape)
    start = _second_start(rows, cols)
    x8 = _empty_act8(x, x.shape, rows, cols, start + 4 * rows - rows * (-(-cols // BLOCK)) * (BLOCK + 1))
    y8 = _empty_act8(x, x.shape, rows, cols) if checkpoint_output else None
    yc, ys = _ptrs(y8) if y8 is not None else (None, None)
    N.check(N.lib().aw4_rms_norm_forward(src.data_ptr(), code, rows, cols, ld, weight.data_ptr(),
                                         N.DTYPE_CODES[weight.dtype], eps, y.data_ptr(), x8.data.data_ptr() + start,
                                         *_ptrs(x8), yc, ys, dev, N.stream_of(dev)), "aw4_rms_norm_forward")
    return y, RMSNormSaved(x8, y8)


def rms_norm_backward(dy: torch.Tensor, weight: torch.Tensor,
                      saved: RMSNormSaved) -> tuple[torch.Tensor, torch.Tensor]:
    """(dx, dweight) from the checkpoint of x; dweight in the weight's dtype."""
    x8 = saved.x8
    _same(dy, x8.device, x8.dtype, "rms_norm_backward: dy")
    if dy.shape != x8.shape:
        raise ValueError(f"rms_norm_backward: dy of shape {tuple(x8.shape)} expected, found {tuple(dy.shape)}")
    src, rows, cols, ld = _rows_of(dy, "rms_norm_backward")
    weight = _check_weight(weight, cols, x8.dtype, x8.device, "rms_norm_backward")
    dev = dy.get_device()
    dx = dy.new_empty(dy.shape)
    dw = torch.empty_like(weight)
    code = N.DTYPE_CODES[dy.dtype]
    nbytes = _norm_workspace(rows, cols, dev)
    ws = dy.new_empty(nbytes, dtype=torch.uint8)
    N.check(N.lib().aw4_rms_norm_backward(src.data_ptr(), code, rows, cols, ld, *_ptrs(x8),
                                          x8.data.data_ptr() + _second_start(rows, cols), weight.data_ptr(),
                                          N.DTYPE_CODES[weight.dtype], dx.data_ptr(), dw.data_ptr(),
                                          ws.data_ptr(), nbytes, dev, N.stream_of(dev)), "aw4_rms_norm_backward")
    return dx, dw


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, checkpoint_output):
        y, saved = rms_norm_forward(x, weight, eps, checkpoint_output=checkpoint_output)
        ctx.save_for_backward(weight, saved.x8.data)
        ctx.x8 = (saved.x8.shape, saved.x8.dtype)
        y8 = saved.output.data if checkpoint_output else None
        if y8 is not None:
            ctx.mark_non_differentiable(y8)
        return y, y8

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, _):
        weight, data = ctx.saved_tensors
        dx, dw = rms_norm_backward(dy, weight, RMSNormSaved(Act8(data, *ctx.x8)))
        return dx, dw, None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *, checkpoint_output: bool = False):
    """Differentiable RMS norm over the last axis that keeps 8 bits of its input.  With
    ``checkpoint_output`` returns (y, checkpoint of y)."""
    y, y8 = _RMSNorm.apply(x, weight, eps, checkpoint_output)
    return (y, Act8(y8, y.shape, y.dtype)) if checkpoint_output else y


# ---------------------------------------------------------------------------
# gated activation
# ---------------------------------------------------------------------------

def swiglu_forward(gate: torch.Tensor, up: torch.Tensor | None = None, *,
                   checkpoint_output: bool = False) -> tuple[torch.Tensor, SwiGLUSaved]:
    """h = gate sigmoid(gate) up, and what the backward call needs.  Without ``up``, ``gate`` holds both
    as halves of its last axis, gate first."""
    code = _dtype_code(gate, "swiglu")
    packed = up is None
    src, rows, cols, ld = _rows_of(gate, "swiglu")
    if packed:
        if cols % 2:
            raise ValueError(f"swiglu: gate and up as halves of the last axis expected, found {cols} columns")
        cols //= 2
        shape = (*gate.shape[:-1], cols)
        other, ld_up = src.data_ptr() + cols * src.element_size(), ld
    else:
        _same(up, gate.device, gate.dtype, "swiglu: up")
        if up.shape != gate.shape:
            raise ValueError(f"swiglu: up of shape {tuple(gate.shape)} expected, found {tuple(up.shape)}")
        shape = gate.shape
        up, _, _, ld_up = _rows_of(up, "swiglu")
        other = up.data_ptr()
    dev = gate.get_device()
    h = gate.new_empty(shape)
    start = _second_start(rows, cols)
    g8 = _empty_act8(gate, shape, rows, cols, start)         # both in one buffer
    u8 = _second_act8(g8, start)
    h8 = _empty_act8(gate, shape, rows, cols) if checkpoint_output else None
    hc, hs = _ptrs(h8) if h8 is not None else (None, None)
    N.check(N.lib().aw4_swiglu_forward(src.data_ptr(), other, code, rows, cols, ld, ld_up, h.data_ptr(),
                                       *_ptrs(g8), *_ptrs(u8), hc, hs, dev, N.stream_of(dev)), "aw4_swiglu_forward")
    return h, SwiGLUSaved(g8, u8, packed, h8)


def swiglu_backward(dh: torch.Tensor, saved: SwiGLUSaved):
    """(dgate, dup) from the checkpoints, or one tensor of both halves where gate and up came as one."""
    g8 = saved.gate8
    _same(dh, g8.device, g8.dtype, "swiglu_backward: dh")
    if dh.shape != g8.shape:
        raise ValueError(f"swiglu_backward: dh of shape {tuple(g8.shape)} expected, found {tuple(dh.shape)}")
    src, rows, cols, ld = _rows_of(dh, "swiglu_backward")
    dev = dh.get_device()
    if saved.packed:
        both = dh.new_empty((*dh.shape[:-1], 2 * cols))
        out, ld_out = both, 2 * cols
        dgate, dup = both.data_ptr(), both.data_ptr() + cols * both.element_size()
    else:
        out = dh.new_empty(dh.shape), dh.new_empty(dh.shape)
        ld_out = cols
        dgate, dup = out[0].data_ptr(), out[1].data_ptr()
    N.check(N.lib().aw4_swiglu_backward(src.data_ptr(), N.DTYPE_CODES[dh.dtype], rows, cols, ld, *_ptrs(g8),
                                        *_ptrs(saved.up8), dgate, dup, ld_out, dev, N.stream_of(dev)),
            "aw4_swiglu_backward")
    return out


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, checkpoint_output):
        h, saved = swiglu_forward(gate, up, checkpoint_output=checkpoint_output)
        ctx.save_for_backward(saved.gate8.data)
        ctx.act8, ctx.packed, ctx.start = (saved.gate8.shape, saved.gate8.dtype), saved.packed, saved.up8.start
        h8 = saved.output.data if checkpoint_output else None
        if h8 is not None:
            ctx.mark_non_differentiable(h8)
        return h, h8

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, _):
        data, = ctx.saved_tensors
        saved = SwiGLUSaved(Act8(data, *ctx.act8), Act8(data, *ctx.act8, ctx.start), ctx.packed)
        out = swiglu_backward(dh, saved)
        return (out, None, None) if ctx.packed else (*out, None)


def swiglu(gate: torch.Tensor, up: torch.Tensor | None = None, *, checkpoint_output: bool = False):
    """Differentiable gated activation that keeps 8 bits of gate and up.  With ``checkpoint_output``
    returns (h, checkpoint of h)."""
    h, h8 = _SwiGLU.apply(gate, up, checkpoint_output)
    return (h, Act8(h8, h.shape, h.dtype)) if checkpoint_output else h


# ---------------------------------------------------------------------------
# projections
# ---------------------------------------------------------------------------

@functools.lru_cache(maxsize=1024)
def _wgrad_workspace(rows: int, n: int, k: int, groups: int, device: int) -> int:
    return int(N.lib().aw4_weight_grad_workspace(rows, n, k, groups, device))


def weight_grad(dy: torch.Tensor, x8: Act8, offsets: torch.Tensor | None = None, *,
                out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
                accumulate: bool = False) -> torch.Tensor:
    """dW = dy^T x from the checkpoint of x: [n, k] for dy [..., n] and x [..., k], bfloat16 or float16,
    summed in float32.

    ``offsets`` (int32, on the device, ascending from 0 to the number of rows) cuts the rows into
    groups; the result is then [groups, n, k] with group g summed over rows offsets[g] to
    offsets[g + 1].  Values outside the rows are cut to them.  The result is in dy's dtype, or
    float32 by ``out_dtype`` or ``out``; with ``accumulate`` it is added to ``out``.
    """
    if dy.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"weight_grad: bfloat16 or float16 expected, found {dy.dtype}")
    _same(dy, x8.device, x8.dtype, "weight_grad: dy")
    if dy.dim() == 0 or dy.shape[:-1] != x8.shape[:-1]:
        raise ValueError(f"weight_grad: dy {tuple(dy.shape)} and the checkpoint {tuple(x8.shape)} differ in rows")
    src, rows, n, ld = _rows_of(dy, "weight_grad")
    k, dev, groups = x8.cols, dy.get_device(), 1
    shape = (n, k)
    if offsets is not None:
        _same(offsets, dy.device, torch.int32, "weight_grad: offsets")
        if offsets.dim() != 1 or offsets.numel() < 2:
            raise ValueError(f"weight_grad: offsets of groups + 1 values expected, found {tuple(offsets.shape)}")
        offsets = offsets.contiguous()
        groups = offsets.numel() - 1
        shape = (groups, n, k)
    if out is None:
        if accumulate:
            raise ValueError("weight_grad: accumulate needs out")
        out = dy.new_empty(shape, dtype=out_dtype or dy.dtype)
    else:
        _same(out, dy.device, out_dtype, "weight_grad: out")
        if out.shape != shape or not out.is_contiguous():
            raise ValueError(f"weight_grad: contiguous out of shape {shape} expected, found {tuple(out.shape)}")
    if out.dtype not in (dy.dtype, torch.float32):
        raise TypeError(f"weight_grad: result in {dy.dtype} or float32 expected, found {out.dtype}")
    if rows and (ld < n or ld % 8 or src.data_ptr() % 16):
        # the bulk copies want rows on 16 bytes
        padded = dy.new_empty((rows, -(-n // 8) * 8))
        padded[:, :n].copy_(src.reshape(rows, n))
        src, ld = padded, padded.shape[1]
    nbytes = _wgrad_workspace(rows, n, k, groups, dev)
    ws = dy.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    N.check(N.lib().aw4_weight_grad(src.data_ptr(), N.DTYPE_CODES[dy.dtype], rows, n, ld, *_ptrs(x8), k,
                                    N.ptr(offsets), groups, out.data_ptr(), N.DTYPE_CODES[out.dtype],
                                    int(accumulate), N.ptr(ws), nbytes, N.wait_status(dev), dev, N.stream_of(dev)),
            "aw4_weight_grad")
    return out


def check_weight_grads(device: torch.device | int | str | None = None, *, synchronize: bool = True) -> None:
    """Raises ``NativeError`` where a weight gradient on this device (the current one) gave up a wait, and forgets
    it.  ``synchronize`` first waits for the device; without it only what has run so far is seen.  The next
    ``weight_grad`` on the device and an optimizer's ``step`` look too, without waiting: a program that uses gradients
    elsewhere, or replays them from a CUDA graph, calls this before it relies on them."""
    if isinstance(device, str):
        device = torch.device(device)
    index = device if isinstance(device, int) else device.index if device is not None else None
    if index is None:
        index = torch.cuda.current_device()
    if synchronize:
        torch.cuda.synchronize(index)
    N.raise_given_up(index)


def _check_linear(x: torch.Tensor, weight: torch.Tensor, x8: Act8 | None, what: str) -> None:
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{what}: bfloat16 or float16 expected, found {x.dtype}")
    N.require_cuda(x, what)
    _same(weight, x.device, x.dtype, f"{what}: weight")
    if x.dim() == 0 or weight.shape[-1] != x.shape[-1]:
        raise ValueError(f"{what}: x {tuple(x.shape)} and weight {tuple(weight.shape)} differ in their last axis")
    if x8 is not None and (x8.shape != x.shape or x8.dtype != x.dtype or x8.device != x.device):
        raise ValueError(f"{what}: the checkpoint {x8} is not one of x {tuple(x.shape)}")


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, x8):
        if x8 is None and ctx.needs_input_grad[1]:
            x8 = quantize_act8(x)
        ctx.save_for_backward(weight, x8.data if ctx.needs_input_grad[1] else None)
        ctx.x8 = (x.shape, x.dtype, x8.start if x8 is not None else 0)
        return torch.nn.functional.linear(x, weight, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, data = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        dx = dy @ weight if need_x else None
        dw = weight_grad(dy, Act8(data, *ctx.x8)) if need_w else None
        db = dy.reshape(-1, dy.shape[-1]).sum(0) if need_b else None
        return dx, dw, db, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
           x8: Act8 | None = None) -> torch.Tensor:
    """Differentiable x W^T + b that keeps 8 bits of x for the weight's gradient.  ``x8``: a checkpoint of
    x that a ``rms_norm`` or ``swiglu`` has already written, kept in place of a new one."""
    _check_linear(x, weight, x8, "linear")
    if weight.dim() != 2:
        raise ValueError(f"linear: weight of two dimensions expected, found {tuple(weight.shape)}")
    return _Linear.apply(x, weight, bias, x8)


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets, x8):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("grouped_linear: reads its offsets on the host, which a CUDA graph cannot capture")
        # cut to the rows, as the weight gradient's kernel cuts them
        ctx.bounds = [min(max(o, 0), x.shape[0]) for o in offsets.tolist()]
        if any(b < a for a, b in zip(ctx.bounds, ctx.bounds[1:])):
            raise ValueError("grouped_linear: offsets that ascend expected: a row belongs to one group")
        if x8 is None and ctx.needs_input_grad[1]:
            x8 = quantize_act8(x)
        ctx.save_for_backward(weight, offsets, x8.data if ctx.needs_input_grad[1] else None)
        ctx.x8 = (x.shape, x.dtype, x8.start if x8 is not None else 0)
        y = x.new_zeros(x.shape[0], weight.shape[1])
        for g, (a, b) in enumerate(zip(ctx.bounds, ctx.bounds[1:])):
            if b > a:
                torch.mm(x[a:b], weight[g].t(), out=y[a:b])
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, offsets, data = ctx.saved_tensors
        need_x, need_w = ctx.needs_input_grad[:2]
        dx = None
        if need_x:
            dx = dy.new_zeros(ctx.x8[0])
            for g, (a, b) in enumerate(zip(ctx.bounds, ctx.bounds[1:])):
                if b > a:
                    torch.mm(dy[a:b], weight[g], out=dx[a:b])
        dw = weight_grad(dy, Act8(data, *ctx.x8), offsets) if need_w else None
        return dx, dw, None, None


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, *,
                   x8: Act8 | None = None) -> torch.Tensor:
    """Differentiable x_g W_g^T over groups of rows: x [rows, k], weight [groups, n, k], offsets int32
    [groups + 1] on the device, ascending from 0 to rows (values outside the rows are cut to them; a row of no
    group gives zeros).  Keeps 8 bits of x; all groups' weight
    gradients are one launch.  The products of the forward pass and of dx are one library product a
    group, for which the offsets are read once on the host (a synchronisation; a CUDA graph cannot capture it)."""
    _check_linear(x, weight, x8, "grouped_linear")
    if x.dim() != 2 or weight.dim() != 3:
        raise ValueError(f"grouped_linear: x [rows, k] and weight [groups, n, k] expected, found "
                         f"{tuple(x.shape)} and {tuple(weight.shape)}")
    _same(offsets, x.device, torch.int32, "grouped_linear: offsets")
    if offsets.shape != (weight.shape[0] + 1,):
        raise ValueError(f"grouped_linear: {weight.shape[0] + 1} offsets expected, found {tuple(offsets.shape)}")
    return _GroupedLinear.apply(x, weight, offsets, x8)
