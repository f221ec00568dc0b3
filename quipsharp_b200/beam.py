"""Beam search: the selection of a step.

`beam_select` picks the best n continuations over beams x vocabulary in one
pass over the logits; `kv_cache.fork_pages` (or PagedKVCache.fork) then reorders
the beams' caches by the parents it returns.
"""
from __future__ import annotations

import torch
from torch import Tensor

from . import _native as N
from .kv_cache import _device_of


def beam_select(logits: Tensor, scores: Tensor, n: int | None = None, finished: Tensor | None = None,
                pad: int = 0) -> tuple[Tensor, Tensor, Tensor]:
    """The best n (default: as many as beams) of each search's continuations by
    scores[b] + log_softmax(logits[b])[token].

    logits (batch, beams, vocab) float32 / float16 / bfloat16, the vocabulary
    contiguous; scores (batch, beams) float32.  A beam's tokens rank by logit
    (ties: the lower token first); the beams' lists merge by score (ties: the
    lower beam first).  NaN logits and scores count as -inf.  finished (batch,
    beams) bool: an ended beam has one continuation, `pad`, with its score as it
    is.  Returns (scores float32, parents int32, tokens int32), each (batch, n);
    parents are beam numbers within the search."""
    got = N.fast().beam_select(logits, scores, n, finished, pad)
    if got is not None:
        return got
    N.refuse_grad("beam_select", logits, scores)
    if not -(1 << 31) <= pad < 1 << 31:
        raise ValueError(f"pad must be an int32, got {pad}")
    dev = _device_of(logits, scores, finished)
    if not N.is_current(dev):
        with torch.cuda.device(dev):
            return beam_select(logits, scores, n, finished, pad)
    dtype = N.IO_DTYPES.get(logits.dtype)
    if dtype is None:
        raise TypeError(f"beam_select: unsupported logits dtype {logits.dtype}")
    if logits.dim() != 3:
        raise ValueError(f"logits must be (batch, beams, vocab), got {tuple(logits.shape)}")
    batch, beams, vocab = logits.shape
    if n is None:
        n = beams
    if scores.dtype is not torch.float32 or (finished is not None and finished.dtype not in (torch.bool, torch.uint8)):
        raise TypeError("scores must be float32 and finished bool")
    if scores.shape != (batch, beams) or (finished is not None and finished.shape != (batch, beams)):
        raise ValueError(f"scores and finished must be ({batch}, {beams})")
    if not 1 <= n <= vocab:
        raise ValueError(f"n must be between 1 and the vocabulary, got {n} of {vocab}")
    strides = logits.stride()
    if strides[2] != 1:
        logits = logits.contiguous()
        strides = logits.stride()
    scores = scores.contiguous()
    if finished is not None:
        finished = finished.contiguous()
    nb = N.workspace_bytes("qs_beam_workspace_bytes", batch, beams, vocab, n)
    if nb < 0:
        raise NotImplementedError(f"beam_select takes up to 64 beams and n up to 64, got {beams} and {n}")
    ws = scores.new_empty((nb + 3) // 4)
    out = scores.new_empty((batch, n))
    picks = scores.new_empty((2, batch, n), dtype=torch.int32)
    at = picks.data_ptr()
    N.check(N.lib().qs_beam_select(logits.data_ptr(), dtype, strides[0], strides[1], batch, beams, vocab,
                                   scores.data_ptr(), None if finished is None else finished.data_ptr(), n, pad,
                                   out.data_ptr(), at, at + 4 * batch * n, ws.data_ptr(), nb, N.raw_stream(dev)))
    return out, *picks.unbind(0)
