"""Paged KV cache operators over torch tensors (include/cq35.h): pages, positions
and slots of a round (`page_plan`), head norm + rotation of its projections with
keys and values written to their slots (`paged_prepare`), attention of the new
tokens over the pages (`paged_attention`).

Tensors lie on one GPU, which need not be the current one; work goes to that
device's current torch stream, or to `stream` (a torch.cuda.Stream). Nothing
waits for the GPU, and every call may be captured into a graph. A cache is a
pair of BF16 tensors [pages, page_size, kv_heads, head_dim] (views with other
strides included, head_dim contiguous).
"""
from __future__ import annotations

import ctypes
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


def _tensor(name, t, dtype, dim, device=None):
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
    return t


def _flat(name, t, dtype, count, device):
    _tensor(name, t, dtype, 1, device)
    if t.shape[0] != count:
        raise ValueError(f"{name} must have {count} entries, not {t.shape[0]}")
    if count > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")
    return t


def _stream(device, stream):
    s = torch.cuda.current_stream(device) if stream is None else stream
    if s.device != device:
        raise ValueError(f"the stream is {s.device}'s, the tensors {device}'s")
    return s


def _heads(name, t, rows, heads, head_dim, device):
    _tensor(name, t, torch.bfloat16, 3, device)
    if tuple(t.shape) != (rows, heads, head_dim):
        raise ValueError(f"{name} must be {(rows, heads, head_dim)}, not {tuple(t.shape)}")
    if t.stride(2) != 1:
        raise ValueError(f"{name}: the channels of a head must be contiguous")
    # the stride of a dimension of length one addresses nothing
    return _lib.Heads(t.data_ptr(), t.stride(0) if rows > 1 else 0, t.stride(1) if heads > 1 else 0)


def _cache(key_cache, value_cache):
    _tensor("key_cache", key_cache, torch.bfloat16, 4)
    _tensor("value_cache", value_cache, torch.bfloat16, 4, key_cache.device)
    if key_cache.shape != value_cache.shape:
        raise ValueError(f"key_cache {tuple(key_cache.shape)} and value_cache {tuple(value_cache.shape)} differ")
    if 0 in key_cache.shape:
        raise ValueError("an empty cache")
    strides = []
    for i in range(3):
        if key_cache.shape[i] > 1 and key_cache.stride(i) != value_cache.stride(i):
            raise ValueError("key_cache and value_cache have different strides")
        strides.append(key_cache.stride(i) if key_cache.shape[i] > 1 else 0)
    if key_cache.stride(3) != 1 or value_cache.stride(3) != 1:
        raise ValueError("the channels of a cached head must be contiguous")
    pages, page_size, kv_heads, head_dim = key_cache.shape
    return _lib.PagedCache(key_cache.data_ptr(), value_cache.data_ptr(), pages, page_size, kv_heads, head_dim, *strides)


def _table(table, requests, device):
    _tensor("table", table, torch.int32, 2, device)
    if requests is not None and table.shape[0] != requests:
        raise ValueError(f"table must have {requests} rows, not {table.shape[0]}")
    if table.shape[1] > 1 and table.stride(1) != 1:
        raise ValueError("the entries of a table row must be contiguous")
    return table.stride(0) if table.shape[0] > 1 else table.shape[1]


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
    device = _tensor("table", table, torch.int32, 2).device
    requests = table.shape[0]
    stride = _table(table, None, device)
    _flat("cached", cached, torch.int32, requests, device)
    _flat("lengths", lengths, torch.int32, requests, device)
    _tensor("free_pages", free_pages, torch.int32, 1, device)
    _flat("free_pages", free_pages, torch.int32, free_pages.shape[0], device)
    _flat("free_count", free_count, torch.int32, 1, device)
    rows = int(rows)
    if rows < 0:
        raise ValueError(f"rows must not be negative: {rows}")
    s = _stream(device, stream)
    if out is None:
        with torch.cuda.stream(s):
            sizes = (requests + 1, rows, rows, 1, 2)
            whole = torch.empty(sum(sizes), dtype=torch.int32, device=device)
            out = PagePlan(*whole.split(sizes))
    else:
        for name, t, n in zip(PagePlan._fields, out, (requests + 1, rows, rows, 1, 2)):
            _flat("out." + name, t, torch.int32, n, device)
    check(_lib.load().cq35_page_plan(
        table.data_ptr(), stride, requests, table.shape[1], cached.data_ptr(), lengths.data_ptr(),
        free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(), page_size, rows, out.row_start.data_ptr(),
        out.positions.data_ptr(), out.slots.data_ptr(), out.free_left.data_ptr(), out.status.data_ptr(), s.cuda_stream))
    return out


def paged_prepare(q, k, v, q_weight, k_weight, inv_freq, positions, slots, key_cache, value_cache, *, eps=1e-6,
                  pair_axis=None, out=None, stream=None):
    """Head norm and rotation of a round's projections (cq35_paged_prepare):
    returns the rotated queries, writes keys and values to cache rows `slots`
    (int32 [rows]; a negative one skips its row, query included). q [rows,
    q_heads, head_dim], k and v [rows, kv_heads, head_dim] BF16 with any row and
    head strides (the query half of a query/gate projection is such a view);
    weights F32 [head_dim]; inv_freq F32 [rope_dim / 2]; positions int32 [rows],
    or [axes, rows] with pair_axis[i] the axis of rotated pair i. `out`: the
    tensor for the queries, q itself allowed."""
    cache = _cache(key_cache, value_cache)
    device = key_cache.device
    _tensor("q", q, torch.bfloat16, 3, device)
    rows, q_heads = q.shape[0], q.shape[1]
    if q_heads == 0:
        raise ValueError("q has no heads")
    hq = _heads("q", q, rows, q_heads, cache.head_dim, device)
    hk = _heads("k", k, rows, cache.kv_heads, cache.head_dim, device)
    hv = _heads("v", v, rows, cache.kv_heads, cache.head_dim, device)
    _flat("q_weight", q_weight, torch.float32, cache.head_dim, device)
    _flat("k_weight", k_weight, torch.float32, cache.head_dim, device)
    _tensor("inv_freq", inv_freq, torch.float32, 1, device)
    pairs = inv_freq.shape[0]
    _flat("inv_freq", inv_freq, torch.float32, pairs, device)
    if positions.dim() == 1:
        positions = positions.unsqueeze(0)
    _tensor("positions", positions, torch.int32, 2, device)
    axes = positions.shape[0]
    if positions.shape[1] != rows or (rows > 1 and positions.stride(1) != 1):
        raise ValueError(f"positions must be [axes, {rows}] with contiguous rows, not {tuple(positions.shape)}")
    _flat("slots", slots, torch.int32, rows, device)
    if pair_axis is not None:
        if len(pair_axis) != pairs or not all(0 <= int(x) < axes for x in pair_axis):
            raise ValueError(f"pair_axis must name one of {axes} axes for each of {pairs} pairs")
        pair_axis = (ctypes.c_uint8 * pairs)(*[int(x) for x in pair_axis])
    s = _stream(device, stream)
    if out is None:
        with torch.cuda.stream(s):
            out = torch.empty((rows, q_heads, cache.head_dim), dtype=torch.bfloat16, device=device)
    ho = _heads("out", out, rows, q_heads, cache.head_dim, device)
    check(_lib.load().cq35_paged_prepare(
        ctypes.byref(cache), ctypes.byref(hq), ctypes.byref(hk), ctypes.byref(hv), rows, q_heads, q_weight.data_ptr(),
        k_weight.data_ptr(), eps, inv_freq.data_ptr(), 2 * pairs, positions.data_ptr(),
        positions.stride(0) if axes > 1 else rows, axes, pair_axis, slots.data_ptr(), ctypes.byref(ho), s.cuda_stream))
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
    cache = _cache(key_cache, value_cache)
    device = key_cache.device
    _tensor("q", q, torch.bfloat16, 3, device)
    rows, q_heads = q.shape[0], q.shape[1]
    if q_heads == 0:
        raise ValueError("q has no heads")
    hq = _heads("q", q, rows, q_heads, cache.head_dim, device)
    hg = None if gate is None else _heads("gate", gate, rows, q_heads, cache.head_dim, device)
    requests = _tensor("lengths", lengths, torch.int32, 1, device).shape[0]
    _flat("lengths", lengths, torch.int32, requests, device)
    _flat("row_start", row_start, torch.int32, requests + 1, device)
    stride = _table(table, requests, device)
    scale = cache.head_dim ** -0.5 if scale is None else float(scale)
    max_rows, max_keys = int(max_rows), int(max_keys)
    s = _stream(device, stream)
    need = paged_attention_workspace(rows, requests, q_heads, cache.kv_heads, cache.head_dim, max_rows, max_keys)
    if workspace is not None:
        _flat("workspace", workspace, torch.uint8, workspace.shape[0] if workspace.dim() == 1 else -1, device)
    with torch.cuda.stream(s):
        if workspace is None and need:
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
        if out is None:
            out = torch.empty((rows, q_heads, cache.head_dim), dtype=torch.bfloat16, device=device)
    ho = _heads("out", out, rows, q_heads, cache.head_dim, device)
    check(_lib.load().cq35_paged_attention(
        ctypes.byref(cache), ctypes.byref(hq), None if hg is None else ctypes.byref(hg), ctypes.byref(ho), rows, q_heads,
        table.data_ptr(), stride, requests, table.shape[1], row_start.data_ptr(), lengths.data_ptr(), scale, max_rows,
        max_keys, None if workspace is None else workspace.data_ptr(), 0 if workspace is None else workspace.shape[0],
        s.cuda_stream))
    return out


def paged_attention_workspace(rows, requests, q_heads, kv_heads, head_dim, max_rows=0, max_keys=0) -> int:
    """Bytes of workspace that paged_attention needs for these sizes."""
    b = ctypes.c_int64()
    check(_lib.load().cq35_paged_attention_workspace(rows, requests, q_heads, kv_heads, head_dim, max_rows, max_keys,
                                                     ctypes.byref(b)))
    return b.value
