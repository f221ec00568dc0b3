"""Attention of new tokens over a paged key-value cache (see kv_cache).

`decode_attention` answers one new token per row, the form of a decoding step;
`window_attention` many new tokens per row (prompts, chunks of prompts, drafted
tokens), causal.  Both share key heads between query heads, and both take a
sliding window with `sinks` first tokens that stay visible: the token in place i
sees the places j <= i with j > i - window or j < sinks.

Products enter the tensor cores in the cache's 16-bit type and are summed in
float32, as are the softmax's maximum and sum.  There is no backward pass: the
decoding path is inference only, like the quantized layers'.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor

from . import _native as N
from .kv_cache import _device_of, _int32, kv_pool


def _arguments(name, q, k_pages, v_pages, table, lengths, window, sinks, scale):
    N.refuse_grad(name, q, k_pages, v_pages)
    if k_pages.dim() != 4 or table.dim() != 2 or q.dim() != 3:
        raise ValueError(f"{name} takes queries (tokens, heads, dim), one layer's pools (pages, heads, page, dim) "
                         "and a table (rows, width)")
    pool, _, kv_heads, page, dim = kv_pool(k_pages, v_pages)
    if q.dtype is not k_pages.dtype:
        raise TypeError(f"queries must have the cache's type {k_pages.dtype}, got {q.dtype}")
    _, heads, q_dim = q.shape
    if q_dim != dim:
        raise ValueError(f"queries of dimension {q_dim} do not match the cache's {dim}")
    if not kv_heads or heads % kv_heads:
        raise ValueError(f"{heads} query heads do not share {kv_heads} key heads evenly")
    if window is None:
        window = 0
    elif window < 1:
        raise ValueError(f"window must be positive or None, got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    rows, width = table.shape
    return (N.rows_of_8(q), pool, kv_heads, page, rows, width, _int32("table", table, rows, width),
            _int32("lengths", lengths, rows), 1.0 / math.sqrt(dim) if scale is None else float(scale),
            min(int(window), 1 << 62), min(int(sinks), 1 << 62))


def decode_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, *,
                     window: int | None = None, sinks: int = 0, scale: float | None = None,
                     return_lse: bool = False):
    """Attention of each row's newest token.

    q (rows, q_heads, dim) float16 / bfloat16; k_pages, v_pages (pages, kv_heads,
    page, dim) of that type; table (rows, width) and lengths (rows,) int32, the
    lengths counting the new token, whose keys and values are already in the
    cache.  Rows of length 0 give 0.  Returns (rows, q_heads, dim), with
    return_lse also log sum exp of the scaled scores, float32 (rows, q_heads)
    (-inf where a row sees nothing).  Keys that are not seen are not read."""
    got = N.fast().attend(q, k_pages, v_pages, table, lengths, None, window, sinks, scale, return_lse)
    if got is not None:
        return got
    dev = _device_of(q, k_pages, v_pages, table, lengths)
    if not N.is_current(dev):
        with torch.cuda.device(dev):
            return decode_attention(q, k_pages, v_pages, table, lengths, window=window, sinks=sinks, scale=scale,
                                    return_lse=return_lse)
    q, pool, kv_heads, page, rows, width, table, lengths, scale, window, sinks = _arguments(
        "decode_attention", q, k_pages, v_pages, table, lengths, window, sinks, scale)
    tokens, heads, dim = q.shape
    if tokens != rows:
        raise ValueError(f"decode_attention takes one query token per row: {tokens} tokens, {rows} rows")
    nb = N.workspace_bytes("qs_attn_decode_workspace_bytes", rows, heads, kv_heads, dim, page, width, window, sinks)
    nb = max(nb, 0)  # below: sizes that the library refuses, with its reason
    ws = lengths.new_empty(nb // 4) if nb else None
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((rows, heads), dtype=torch.float32) if return_lse else None
    qs = q.stride()
    N.check(N.lib().qs_attn_decode(q.data_ptr(), qs[0], qs[1], pool, rows, heads, width, table.data_ptr(),
                                   lengths.data_ptr(), scale, window, sinks, out.data_ptr(),
                                   lse.data_ptr() if return_lse else None, ws.data_ptr() if nb else None, nb,
                                   N.raw_stream(dev)))
    return (out, lse) if return_lse else out


def window_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, cu: Tensor, *,
                     window: int | None = None, sinks: int = 0, scale: float | None = None,
                     return_lse: bool = False):
    """Causal attention of each row's new tokens.

    q (tokens, q_heads, dim) packed: row r's tokens are [cu[r], cu[r+1]) (cu int32
    (rows + 1,)) and take its last places, which `lengths` counts and whose keys
    and values are already in the cache; everything else as in decode_attention.
    Up to 128 query heads share a key head."""
    got = N.fast().attend(q, k_pages, v_pages, table, lengths, cu, window, sinks, scale, return_lse)
    if got is not None:
        return got
    dev = _device_of(q, k_pages, v_pages, table, lengths, cu)
    if not N.is_current(dev):
        with torch.cuda.device(dev):
            return window_attention(q, k_pages, v_pages, table, lengths, cu, window=window, sinks=sinks, scale=scale,
                                    return_lse=return_lse)
    q, pool, kv_heads, page, rows, width, table, lengths, scale, window, sinks = _arguments(
        "window_attention", q, k_pages, v_pages, table, lengths, window, sinks, scale)
    cu = _int32("cu", cu, rows + 1)
    tokens, heads, dim = q.shape
    nb = N.workspace_bytes("qs_attn_window_workspace_bytes", tokens, rows, heads, kv_heads, dim, page, width, window, sinks)
    nb = max(nb, 0)  # below: sizes that the library refuses, with its reason
    ws = lengths.new_empty(nb // 4) if nb else None
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if return_lse else None
    qs = q.stride()
    N.check(N.lib().qs_attn_window(q.data_ptr(), qs[0], qs[1], pool, tokens, rows, heads, width, table.data_ptr(),
                                   lengths.data_ptr(), cu.data_ptr(), scale, window, sinks, out.data_ptr(),
                                   lse.data_ptr() if return_lse else None, ws.data_ptr() if nb else None, nb,
                                   N.raw_stream(dev)))
    return (out, lse) if return_lse else out
