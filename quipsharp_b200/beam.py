"""Beam search: the selection of a step.

`beam_select` picks the best n continuations over beams x vocabulary in one
pass over the logits; `kv_cache.fork_pages` (or PagedKVCache.fork) then reorders
the beams' caches by the parents it returns.
"""
from __future__ import annotations

import torch
from torch import Tensor

from . import _native as N


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
    N.refuse_grad("beam_select", logits, scores)
    N.require_cuda(logits, scores, finished)
    if logits.dtype not in N.IO_DTYPES:
        raise TypeError(f"beam_select: unsupported logits dtype {logits.dtype}")
    if logits.dim() != 3:
        raise ValueError(f"logits must be (batch, beams, vocab), got {tuple(logits.shape)}")
    batch, beams, vocab = logits.shape
    if n is None:
        n = beams
    if scores.dtype != torch.float32 or (finished is not None and finished.dtype not in (torch.bool, torch.uint8)):
        raise TypeError("scores must be float32 and finished bool")
    if scores.shape != (batch, beams) or (finished is not None and finished.shape != (batch, beams)):
        raise ValueError(f"scores and finished must be ({batch}, {beams})")
    if any(t is not None and t.device != logits.device for t in (scores, finished)):
        raise ValueError("all tensors must be on one device")
    if not 1 <= n <= vocab:
        raise ValueError(f"n must be between 1 and the vocabulary, got {n} of {vocab}")
    if logits.stride(2) != 1:
        logits = logits.contiguous()
    scores = scores.contiguous()
    finished = None if finished is None else finished.contiguous()
    dev = logits.device
    with N.device_guard(dev):
        nb = N.lib().qs_beam_workspace_bytes(batch, beams, vocab, n)
        if nb < 0:
            raise NotImplementedError(f"beam_select takes up to 64 beams and n up to 64, got {beams} and {n}")
        ws = torch.empty(nb, dtype=torch.uint8, device=dev)
        out = torch.empty(batch, n, dtype=torch.float32, device=dev)
        parents, tokens = torch.empty(2, batch, n, dtype=torch.int32, device=dev).unbind(0)
        N.check(N.lib().qs_beam_select(logits.data_ptr(), N.IO_DTYPES[logits.dtype], logits.stride(0), logits.stride(1),
                                       batch, beams, vocab, scores.data_ptr(), N.ptr(finished), n, pad, out.data_ptr(),
                                       parents.data_ptr(), tokens.data_ptr(), ws.data_ptr(), nb,
                                       N.raw_stream(dev.index)))
    return out, parents, tokens
