"""8-bit rows and products over torch tensors (include/cq35.h): rows of 8-bit
integers with a scale each (`quantize_rows`, also of weights, whose outputs are
rows), of a residual's addition and norm (`norm_quantize`), of a gated
feed-forward's product (`gated_quantize`), and the product of two such matrices
(`int8_linear`).

Tensors lie on one GPU, which need not be the current one; work goes to that
device's current torch stream, or to `stream` (a torch.cuda.Stream). Nothing
waits for the GPU, and every call may be captured into a graph. Results carry no
gradients. Rows may lie apart (views of wider tensors), their channels, a
multiple of 16, are contiguous.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from ._lib import check
from .paged import _F32, _flat, _stream, _tensor, _why

_TYPES = {torch.bfloat16: 0, torch.float32: 1}  # CQ35_BF16, CQ35_F32
_I8 = torch.int8


class Int8Rows(NamedTuple):
    data: torch.Tensor   # int8 [rows, channels]
    scale: torch.Tensor  # float32 [rows]: a row stands for data * scale


class NormRows(NamedTuple):
    data: torch.Tensor    # int8 [rows, channels]
    scale: torch.Tensor   # float32 [rows]
    summed: torch.Tensor  # [rows, channels]: x + residual (x itself without one)


def _rows(name, t, shape=None, dtype=None, device=None):
    """A matrix of BF16 or F32 and its description."""
    if not (isinstance(t, torch.Tensor) and t.dim() == 2 and t.is_cuda and t.dtype in _TYPES and
            (dtype is None or t.dtype is dtype) and (device is None or t.device == device)):
        if isinstance(t, torch.Tensor) and dtype is None and t.dtype not in _TYPES:
            raise ValueError(f"{name} must be torch.bfloat16 or torch.float32, not {t.dtype}")
        _why(name, t, t.dtype if dtype is None and isinstance(t, torch.Tensor) else dtype, 2, device)
    rows, channels = t.shape
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, not {tuple(t.shape)}")
    row, channel = t.stride()
    if channel != 1 and channels > 1:
        raise ValueError(f"{name}: the channels of a row must be contiguous")
    # the stride of a dimension of length one addresses nothing
    return _lib.Rows(t.data_ptr(), row if rows > 1 else 0, _TYPES[t.dtype])


def _int8_rows(name, r, device=None):
    """An 8-bit matrix with its scales, its shape and its description."""
    try:
        data, scale = r[0], r[1]
    except (TypeError, IndexError, KeyError):
        raise TypeError(f"{name} must be a pair of 8-bit rows and their scales") from None
    rows, channels = _tensor(name, data, _I8, 2, device).shape
    row, channel = data.stride()
    if channel != 1 and channels > 1:
        raise ValueError(f"{name}: the channels of a row must be contiguous")
    return data, rows, channels, _lib.Int8Rows(data.data_ptr(), row if rows > 1 else 0,
                                               _flat(name + " scales", scale, _F32, rows, data.device))


def _output(out, like, rows, channels, under):
    """Where 8-bit rows go: new tensors, or the caller's."""
    if out is None:
        with under:
            data, scale = like.new_empty((rows, channels), dtype=_I8), like.new_empty(rows, dtype=_F32)
        return data, scale, _lib.Int8Rows(data.data_ptr(), channels, scale.data_ptr())
    data, have, width, described = _int8_rows("out", out, like.device)
    if have != rows or width != channels:
        raise ValueError(f"out must be {(rows, channels)}, not {(have, width)}")
    return data, out[1], described


def quantize_rows(x, *, out=None, stream=None) -> Int8Rows:
    """Each row of x (BF16 or F32 [rows, channels]) as 8-bit integers with a scale
    of its own, the row's largest magnitude over 127 (cq35_quantize_rows). `out`: a
    pair of tensors to write to."""
    hx = _rows("x", x)
    rows, channels = x.shape
    raw, under = _stream(x.device, stream)
    data, scale, ho = _output(out, x, rows, channels, under)
    check(_lib.load().cq35_quantize_rows(hx, rows, channels, ho, raw))
    return Int8Rows(data, scale)


def norm_quantize(x, weight, *, residual=None, eps=1e-6, summed=None, out=None, stream=None) -> NormRows:
    """The norm h * weight / sqrt(mean(h^2) + eps) of h = x + residual as 8-bit rows,
    and h itself (cq35_norm_quantize). x and residual BF16 or F32 [rows, channels],
    weight F32 [channels]. h is rounded to their type; without a residual it is x.
    `summed`: the tensor for h, x or residual itself allowed; `out`: a pair of
    tensors for the 8-bit rows."""
    hx = _rows("x", x)
    rows, channels = shape = x.shape
    device = x.device
    weight = _flat("weight", weight, _F32, channels, device)
    raw, under = _stream(device, stream)
    hr = hs = None
    if residual is None:
        if summed is not None and summed is not x:
            raise ValueError("summed is x itself without a residual")
        summed = x
    else:
        hr = _rows("residual", residual, shape, x.dtype, device)
        if summed is None:
            with under:
                summed = x.new_empty(shape)
            hs = _lib.Rows(summed.data_ptr(), channels, hx.dtype)
        else:
            hs = _rows("summed", summed, shape, x.dtype, device)
    data, scale, ho = _output(out, x, rows, channels, under)
    check(_lib.load().cq35_norm_quantize(hx, hr, weight, eps, rows, channels, hs, ho, raw))
    return NormRows(data, scale, summed)


def gated_quantize(gate, up, *, out=None, stream=None) -> Int8Rows:
    """gate * sigmoid(gate) * up as 8-bit rows (cq35_gated_quantize); gate and up
    BF16 or F32 [rows, channels], the halves of one projection's rows for instance.
    `out`: a pair of tensors to write to."""
    hg = _rows("gate", gate)
    rows, channels = shape = gate.shape
    hu = _rows("up", up, shape, gate.dtype, gate.device)
    raw, under = _stream(gate.device, stream)
    data, scale, ho = _output(out, gate, rows, channels, under)
    check(_lib.load().cq35_gated_quantize(hg, hu, rows, channels, ho, raw))
    return Int8Rows(data, scale)


def int8_linear(x, w, *, dtype=torch.bfloat16, out=None, stream=None):
    """The product of 8-bit rows x (a pair of data [rows, channels] and scales, what
    the operators above return) with weights w (a pair of [outputs, channels] and a
    scale for each output): [rows, outputs] of `dtype` (BF16 or F32), the sums exact
    (cq35_int8_linear). `out`: the tensor for it, whose type then counts."""
    data, rows, channels, hx = _int8_rows("x", x)
    device = data.device
    _, outputs, width, hw = _int8_rows("w", w, device)
    if width != channels:
        raise ValueError(f"x has {channels} channels, w {width}")
    raw, under = _stream(device, stream)
    if out is None:
        kind = _TYPES.get(dtype)
        if kind is None:
            raise ValueError(f"dtype must be torch.bfloat16 or torch.float32, not {dtype}")
        with under:
            out = data.new_empty((rows, outputs), dtype=dtype)
        ho = _lib.Rows(out.data_ptr(), outputs, kind)
    else:
        ho = _rows("out", out, (rows, outputs), None, device)
        ho.row_stride = max(ho.row_stride, outputs) if rows <= 1 else ho.row_stride
    check(_lib.load().cq35_int8_linear(hx, hw, rows, outputs, channels, ho, raw))
    return out
