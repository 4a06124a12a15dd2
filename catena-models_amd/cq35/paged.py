"""Paged KV cache operators over torch tensors (include/cq35.h): pages, positions
and slots of a round (`page_plan`), head norm + rotation of its projections with
keys and values written to their slots (`paged_prepare`), attention of the new
tokens over the pages (`paged_attention`).

Tensors lie on one GPU, which need not be the current one; work goes to that
device's current torch stream, or to `stream` (a torch.cuda.Stream). Nothing
waits for the GPU, and every call may be captured into a graph. Results carry no
gradients. Rows of a result that the call leaves alone (no slot, no request) are
uninitialised where the result is new: a round of more rows than its requests
have, whose rows all go on into other work, passes an `out` zeroed beforehand. A
cache is a pair of BF16 tensors [pages, page_size, kv_heads, head_dim] (views
with other strides included, head_dim contiguous).
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import operator
from typing import NamedTuple

import torch

from . import _lib
from ._lib import check


class PagePlan(NamedTuple):
    row_start: torch.Tensor  # int32 [requests + 1]: first row of each request
    positions: torch.Tensor  # int32 [rows]
    slots: torch.Tensor      # int32 [rows]: cache row of each new token, -1 behind the last request's
    free_left: torch.Tensor  # int32 [1]: the free pages after the round
    status: torch.Tensor     # int32 [2]: 0 or what went wrong, and how much is missing


PLAN_STATUS = ("ok", "too few free pages", "too few rows", "lengths outside the tables", "malformed stack of free pages")


_I32, _F32, _BF16 = torch.int32, torch.float32, torch.bfloat16


def _why(name, t, dtype, dim, device):
    """Why a tensor was refused: looked for after the cheap checks of a call,
    which take a few tenths of a microsecond each, beside a launch of about 3."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimensions, not {t.dim()}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not {device}")


def _tensor(name, t, dtype, dim, device=None):
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.dim() == dim and
            (t.is_cuda if device is None else t.device == device)):
        _why(name, t, dtype, dim, device)
    return t


def _flat(name, t, dtype, count, device):
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == (count,) and t.device == device and t.is_contiguous():
        return t.data_ptr()
    _why(name, t, dtype, 1, device)
    if t.shape[0] != count:
        raise ValueError(f"{name} must have {count} entries, not {t.shape[0]}")
    raise ValueError(f"{name} must be contiguous")


def _stream(device, stream):
    """The raw stream of a call, and what its new tensors are made under."""
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device.index), _HERE  # a Stream object would take a tenth of the call
    if stream.device != device:
        raise ValueError(f"the stream is {stream.device}'s, the tensors {device}'s")
    return stream.cuda_stream, torch.cuda.stream(stream)


_HERE = contextlib.nullcontext()


def _heads(name, t, shape, device):
    if not (isinstance(t, torch.Tensor) and t.dtype is _BF16 and t.shape == shape and t.device == device):
        _why(name, t, _BF16, 3, device)
        raise ValueError(f"{name} must be {shape}, not {tuple(t.shape)}")
    row, head, channel = t.stride()
    if channel != 1:
        raise ValueError(f"{name}: the channels of a head must be contiguous")
    # the stride of a dimension of length one addresses nothing
    return _lib.Heads(t.data_ptr(), row if shape[0] > 1 else 0, head if shape[1] > 1 else 0)


def _new_like(q, shape):
    """A contiguous tensor like q and its description."""
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    return out, _lib.Heads(out.data_ptr(), shape[1] * shape[2], shape[2])


def _query_shape(q, cache, device):
    """q's shape as it has to be, its rows and its heads."""
    rows, q_heads, _ = _tensor("q", q, _BF16, 3, device).shape
    if q_heads == 0:
        raise ValueError("q has no heads")
    return (rows, q_heads, cache.head_dim), rows, q_heads


def _cache(key_cache, value_cache):
    shape, device = _tensor("key_cache", key_cache, _BF16, 4).shape, key_cache.device
    if not (isinstance(value_cache, torch.Tensor) and value_cache.dtype is _BF16 and value_cache.shape == shape and
            value_cache.device == device):
        _why("value_cache", value_cache, _BF16, 4, device)
        raise ValueError(f"key_cache {tuple(shape)} and value_cache {tuple(value_cache.shape)} differ")
    pages, page_size, kv_heads, head_dim = shape
    if not (pages and page_size and kv_heads and head_dim):
        raise ValueError("an empty cache")
    # the stride of a dimension of length one addresses nothing
    page, row, head, channel = strides = key_cache.stride()
    other = value_cache.stride()
    if channel != 1 or other[3] != 1:
        raise ValueError("the channels of a cached head must be contiguous")
    if strides != other and any(n > 1 and x != y for n, x, y in zip(shape, strides, other)):
        raise ValueError("key_cache and value_cache have different strides")
    return device, _lib.PagedCache(key_cache.data_ptr(), value_cache.data_ptr(), pages, page_size, kv_heads, head_dim,
                           page if pages > 1 else 0, row if page_size > 1 else 0, head if kv_heads > 1 else 0)


def _table(table, requests, device=None):
    """Rows, width and row stride of a block table."""
    count, width = _tensor("table", table, _I32, 2, device).shape
    if requests is not None and count != requests:
        raise ValueError(f"table must have {requests} rows, not {count}")
    row, entry = table.stride()
    if entry != 1 and width > 1:
        raise ValueError("the entries of a table row must be contiguous")
    return count, width, row if count > 1 else width


def _int32(name, x):
    """A number as the library's 32 bits hold it; others would be taken modulo 2^32."""
    x = operator.index(x)
    if not -1 << 31 <= x < 1 << 31:
        raise ValueError(f"{name} is out of range: {x}")
    return x


def _pair_axis(pair_axis, pairs, axes):
    """One byte a pair, from a sequence, an array or a tensor of whole numbers in
    host memory (one on the GPU would be waited for)."""
    try:
        named = bytes(list(pair_axis))  # an array's own bytes are not its values
    except (TypeError, ValueError, OverflowError) as e:
        raise (TypeError if isinstance(e, TypeError) else ValueError)(f"pair_axis must hold whole numbers from 0 to {axes - 1}: {e}") from None
    if len(named) != pairs or not named or max(named) >= axes:
        raise ValueError(f"pair_axis must name one of {axes} axes for each of {pairs} pairs")
    return named


def page_plan(table, cached, lengths, free_pages, free_count, *, page_size, rows, out=None, stream=None) -> PagePlan:
    """Pages, positions and slots of a round (cq35_page_plan): request r holds
    cached[r] tokens and is to hold lengths[r] (int32 [requests]). `table` (int32
    [requests, width]) and the stack `free_pages` (int32 [pages], the first
    free_count[0] of them free) are updated in place; pages given back by
    requests that get shorter are used first. `rows` is the length of
    `positions` and `slots`, at least the sum of the new tokens. `out`: an
    earlier plan's tensors to write to. `status` is for the caller to look at
    when it next waits for the GPU: unless status[0] is 0 (PLAN_STATUS), nothing
    was changed and the round has no rows."""
    if type(page_size) is not int or not 0 < page_size < 1 << 31:
        page_size = _int32("page_size", page_size)
    requests, width, stride = _table(table, None)
    device = table.device
    cached, lengths = _flat("cached", cached, _I32, requests, device), _flat("lengths", lengths, _I32, requests, device)
    pages = free_pages.numel() if isinstance(free_pages, torch.Tensor) else 0
    free_pages = _flat("free_pages", free_pages, _I32, pages, device)
    free_count = _flat("free_count", free_count, _I32, 1, device)
    rows = int(rows)
    if rows < 0:
        raise ValueError(f"rows must not be negative: {rows}")
    raw, under = _stream(device, stream)
    sizes = (requests + 1, rows, rows, 1, 2)
    if out is None:
        with under:
            one = table.new_empty(requests + 2 * rows + 4)
        out = PagePlan(*one.split_with_sizes(sizes))
        base = one.data_ptr()
        at = [base + 4 * n for n in (0, requests + 1, requests + 1 + rows, requests + 1 + 2 * rows, requests + 2 + 2 * rows)]
    else:
        at = [_flat("out." + name, t, _I32, n, device) for name, t, n in zip(PagePlan._fields, out, sizes)]
    check(_lib.load().cq35_page_plan(table.data_ptr(), stride, requests, width, cached, lengths, free_pages, pages, free_count,
                                     page_size, rows, *at, raw))
    return out


def paged_prepare(q, k, v, q_weight, k_weight, inv_freq, positions, slots, key_cache, value_cache, *, eps=1e-6,
                  pair_axis=None, out=None, stream=None):
    """Head norm and rotation of a round's projections (cq35_paged_prepare):
    returns the rotated queries, writes keys and values to cache rows `slots`
    (int32 [rows]; a negative one skips its row, query included). q [rows,
    q_heads, head_dim], k and v [rows, kv_heads, head_dim] BF16 with any row and
    head strides (the query half of a query/gate projection is such a view);
    weights F32 [head_dim]; inv_freq F32 [rope_dim / 2]; positions int32 [rows],
    or [axes, rows] (an expanded row included) with pair_axis[i] (held
    on the host) the axis of rotated pair i. `out`: the tensor for the queries, q itself allowed."""
    device, cache = _cache(key_cache, value_cache)
    shape, rows, q_heads = _query_shape(q, cache, device)
    kv_shape = (rows, cache.kv_heads, cache.head_dim)
    hq, hk, hv = _heads("q", q, shape, device), _heads("k", k, kv_shape, device), _heads("v", v, kv_shape, device)
    q_weight = _flat("q_weight", q_weight, _F32, shape[2], device)
    k_weight = _flat("k_weight", k_weight, _F32, shape[2], device)
    pairs = inv_freq.numel() if isinstance(inv_freq, torch.Tensor) else 0
    inv_freq = _flat("inv_freq", inv_freq, _F32, pairs, device)
    flat = isinstance(positions, torch.Tensor) and positions.dim() == 1
    _tensor("positions", positions, _I32, 1 if flat else 2, device)
    axes, axis_stride = (1, rows) if flat else (positions.shape[0], positions.stride(0))
    if positions.shape[-1] != rows or (rows > 1 and positions.stride(-1) != 1):
        raise ValueError(f"positions must be [axes, {rows}] with contiguous rows, not {tuple(positions.shape)}")
    slots = _flat("slots", slots, _I32, rows, device)
    if pair_axis is not None:
        pair_axis = _pair_axis(pair_axis, pairs, axes)
    raw, under = _stream(device, stream)
    if out is None:
        with under:
            out, ho = _new_like(q, shape)
    else:
        ho = _heads("out", out, shape, device)
    check(_lib.load().cq35_paged_prepare(cache, hq, hk, hv, rows, q_heads, q_weight, k_weight, eps, inv_freq, 2 * pairs,
                                         positions.data_ptr(), axis_stride, axes, pair_axis, slots, ho, raw))
    return out


def paged_attention(q, key_cache, value_cache, table, row_start, lengths, *, gate=None, scale=None, max_rows=0,
                    max_keys=0, out=None, workspace=None, stream=None):
    """Attention of new tokens over a paged cache (cq35_paged_attention): rows
    row_start[r] up to row_start[r + 1] of q [rows, q_heads, head_dim] are the
    last tokens of request r, whose lengths[r] tokens lie in the pages of table
    row r; each row sees the keys up to its own position. `gate` (shaped like q)
    multiplies the result by its sigmoid; `scale` is head_dim^-0.5 by default.
    max_rows and max_keys: what the caller knows of the most rows and keys of any
    request (0: nothing), for the launch alone. `out`: the tensor for the result
    (rows outside every request are left as they were), q itself allowed.
    `workspace`: a uint8 tensor of paged_attention_workspace bytes used by no
    other work at the time, by default allocated for the call."""
    device, cache = _cache(key_cache, value_cache)
    shape, rows, q_heads = _query_shape(q, cache, device)
    hq = _heads("q", q, shape, device)
    hg = None if gate is None else _heads("gate", gate, shape, device)
    requests = lengths.numel() if isinstance(lengths, torch.Tensor) else 0
    lengths = _flat("lengths", lengths, _I32, requests, device)
    row_start = _flat("row_start", row_start, _I32, requests + 1, device)
    _, width, stride = _table(table, requests, device)
    scale = cache.head_dim ** -0.5 if scale is None else float(scale)
    max_rows, max_keys = int(max_rows), int(max_keys)
    raw, under = _stream(device, stream)
    have = at = None
    if workspace is not None:
        have = workspace.numel() if isinstance(workspace, torch.Tensor) else 0
        at = _flat("workspace", workspace, torch.uint8, have, device)
    with under:
        if workspace is None:
            have = paged_attention_workspace(rows, requests, q_heads, cache.kv_heads, cache.head_dim, max_rows, max_keys)
            if have:
                workspace = q.new_empty((have + 1) // 2)
                at = workspace.data_ptr()
        if out is None:
            out, ho = _new_like(q, shape)
        else:
            ho = _heads("out", out, shape, device)
    check(_lib.load().cq35_paged_attention(cache, hq, hg, ho, rows, q_heads, table.data_ptr(), stride, requests, width,
                                           row_start, lengths, scale, max_rows, max_keys, at, have, raw))
    return out


@functools.lru_cache(maxsize=1024)  # of sizes alone
def paged_attention_workspace(rows, requests, q_heads, kv_heads, head_dim, max_rows=0, max_keys=0) -> int:
    """Bytes of workspace that paged_attention needs for these sizes."""
    b = ctypes.c_int64()
    q_heads, kv_heads, head_dim = _int32("q_heads", q_heads), _int32("kv_heads", kv_heads), _int32("head_dim", head_dim)
    check(_lib.load().cq35_paged_attention_workspace(rows, requests, q_heads, kv_heads, head_dim, max_rows, max_keys,
                                                     ctypes.byref(b)))
    return b.value
