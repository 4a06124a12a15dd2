"""Log probabilities over torch tensors (include/cq35.h): of given tokens, with
the entropy of each row of logits and its most likely tokens.

Tensors, streams and capture are as with the other operators (paged.py, int8.py).
"""
from __future__ import annotations

import ctypes
import functools
import operator
from typing import NamedTuple

import torch

from . import _lib
from ._lib import check
from .int8 import _rows
from .paged import _F32, _flat, _stream, _why

_I64, _U8 = torch.int64, torch.uint8


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # float32, shaped like tokens
    entropy: torch.Tensor       # float32 [rows]
    top_tokens: torch.Tensor    # int64 [rows, top], the most likely first
    top_logprobs: torch.Tensor  # float32 [rows, top]


def _results(out, given, rows, top, device):
    if not isinstance(out, (tuple, list)) or len(out) != len(TokenLogprobs._fields):
        raise TypeError("out must be the four tensors of a TokenLogprobs")
    for name, t, shape, dtype in zip(TokenLogprobs._fields, out, (given, (rows,), (rows, top), (rows, top)), (_F32, _F32, _I64, _F32)):
        if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device and t.is_contiguous()):
            _why("out." + name, t, dtype, len(shape), device)
            raise ValueError(f"out.{name} must be contiguous {tuple(shape)}, not {tuple(t.shape)}")


def token_logprobs(logits, tokens, *, top=0, out=None, workspace=None, stream=None) -> TokenLogprobs:
    """Log probabilities (cq35_token_logprobs) under each row of logits (BF16 or F32
    [rows, vocab], rows of any stride) of its tokens (int64 [rows] or [rows, given],
    contiguous), the rows' entropies and their `top` most likely tokens, of equal
    ones the lowest first. A token outside the vocabulary gets NaN, a row that holds
    NaN or +inf or nothing above -inf NaN throughout. `out`: an earlier result's
    tensors to write to; `workspace`: a uint8 tensor of token_logprobs_workspace
    bytes used by no other work at the time, by default allocated for the call."""
    hl = _rows("logits", logits)
    rows, vocab = logits.shape
    device = logits.device
    if not (isinstance(tokens, torch.Tensor) and tokens.dtype is _I64 and tokens.device == device and
            tokens.dim() in (1, 2) and tokens.shape[0] == rows and tokens.is_contiguous()):
        _why("tokens", tokens, _I64, tokens.dim() if isinstance(tokens, torch.Tensor) and tokens.dim() in (1, 2) else 2, device)
        raise ValueError(f"tokens must be {rows} contiguous rows, not {tuple(tokens.shape)}")
    given = 1 if tokens.dim() == 1 else tokens.shape[1]
    if type(top) is not int or not 0 <= top <= 32:
        top = operator.index(top)
        if not 0 <= top <= 32:
            raise ValueError(f"top must be from 0 to 32, not {top}")
    raw, under = _stream(device, stream)
    need = token_logprobs_workspace(rows, vocab, given, top)
    have = at = None
    if workspace is not None:
        have = workspace.numel() if isinstance(workspace, torch.Tensor) else 0
        at = _flat("workspace", workspace, _U8, have, device)
    with under:
        if workspace is None and need:
            workspace = logits.new_empty(need, dtype=_U8)
            at = workspace.data_ptr()
        have = have if have is not None else need
        if out is None:
            # one allocation: the 64-bit tokens in front of the numbers
            whole = logits.new_empty(rows * (3 * top + given + 1), dtype=_F32)
            parts = whole.split_with_sizes((2 * rows * top, rows * top, rows * given, rows))
            out = TokenLogprobs(parts[2].view(tokens.shape), parts[3], parts[0].view(_I64).view(rows, top),
                                parts[1].view(rows, top))
        else:
            _results(out, tokens.shape, rows, top, device)
    check(_lib.load().cq35_token_logprobs(hl, rows, vocab, tokens.data_ptr(), given, top, out[0].data_ptr(), out[1].data_ptr(),
                                          out[2].data_ptr(), out[3].data_ptr(), at, have, raw))
    return TokenLogprobs(*out)


@functools.lru_cache(maxsize=1024)  # of sizes alone
def token_logprobs_workspace(rows, vocab, given=1, top=0) -> int:
    """Bytes of workspace that token_logprobs needs for these sizes."""
    b = ctypes.c_int64()
    check(_lib.load().cq35_token_logprobs_workspace(rows, vocab, given, top, ctypes.byref(b)))
    return b.value
