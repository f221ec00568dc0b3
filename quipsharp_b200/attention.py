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
from .kv_cache import _int32, _same_device, kv_pool


def _arguments(name, q, k_pages, v_pages, table, lengths, window, sinks, scale):
    N.refuse_grad(name, q)
    if k_pages.dim() != 4 or table.dim() != 2 or q.dim() != 3:
        raise ValueError(f"{name} takes queries (tokens, heads, dim), one layer's pools (pages, heads, page, dim) "
                         "and a table (rows, width)")
    pool = kv_pool(k_pages, v_pages)
    if q.dtype != k_pages.dtype:
        raise TypeError(f"queries must have the cache's type {k_pages.dtype}, got {q.dtype}")
    tokens, heads, dim = q.shape
    if dim != pool.dim:
        raise ValueError(f"queries of dimension {dim} do not match the cache's {pool.dim}")
    if heads % pool.heads:
        raise ValueError(f"{heads} query heads do not share {pool.heads} key heads evenly")
    if window is not None and window < 1:
        raise ValueError(f"window must be positive or None, got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    rows, width = table.shape
    return (N.rows_of_8(q), pool, rows, width, _int32("table", table, rows, width), _int32("lengths", lengths, rows),
            1.0 / math.sqrt(dim) if scale is None else float(scale), 0 if window is None else int(window), int(sinks))


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
    _same_device(q, k_pages, v_pages, table, lengths)
    q, pool, rows, width, table, lengths, scale, window, sinks = _arguments(
        "decode_attention", q, k_pages, v_pages, table, lengths, window, sinks, scale)
    if q.shape[0] != rows:
        raise ValueError(f"decode_attention takes one query token per row: {q.shape[0]} tokens, {rows} rows")
    heads = q.shape[1]
    dev = q.device
    with N.device_guard(dev):
        nb = N.lib().qs_attn_decode_workspace_bytes(rows, heads, pool.heads, pool.dim)
        if nb < 0:
            raise NotImplementedError(f"head dimension must be a multiple of 8 up to 128, got {pool.dim}")
        ws = torch.empty(nb, dtype=torch.uint8, device=dev)
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        lse = torch.empty(rows, heads, dtype=torch.float32, device=dev) if return_lse else None
        N.check(N.lib().qs_attn_decode(q.data_ptr(), q.stride(0), q.stride(1), N.ref(pool), rows, heads, width,
                                       table.data_ptr(), lengths.data_ptr(), scale, window, sinks, out.data_ptr(),
                                       N.ptr(lse), ws.data_ptr(), nb, N.raw_stream(dev.index)))
    return (out, lse) if return_lse else out


def window_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, cu: Tensor, *,
                     window: int | None = None, sinks: int = 0, scale: float | None = None,
                     return_lse: bool = False):
    """Causal attention of each row's new tokens.

    q (tokens, q_heads, dim) packed: row r's tokens are [cu[r], cu[r+1]) (cu int32
    (rows + 1,)) and take its last places, which `lengths` counts and whose keys
    and values are already in the cache; everything else as in decode_attention.
    Up to 128 query heads share a key head.  Values that are infinite or NaN are
    only kept from tokens that do not see them where no token of the same tile
    does (places past a row's length never enter)."""
    _same_device(q, k_pages, v_pages, table, lengths, cu)
    q, pool, rows, width, table, lengths, scale, window, sinks = _arguments(
        "window_attention", q, k_pages, v_pages, table, lengths, window, sinks, scale)
    cu = _int32("cu", cu, rows + 1)
    tokens, heads = q.shape[:2]
    dev = q.device
    with N.device_guard(dev):
        nb = N.lib().qs_attn_window_workspace_bytes(tokens, rows, heads, pool.heads, pool.dim)
        if nb < 0:
            raise NotImplementedError(f"head dimension must be a multiple of 8 up to 128, got {pool.dim}")
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        lse = torch.empty(tokens, heads, dtype=torch.float32, device=dev) if return_lse else None
        N.check(N.lib().qs_attn_window(q.data_ptr(), q.stride(0), q.stride(1), N.ref(pool), tokens, rows, heads, width,
                                       table.data_ptr(), lengths.data_ptr(), cu.data_ptr(), scale, window, sinks,
                                       out.data_ptr(), N.ptr(lse), N.ptr(ws), nb, N.raw_stream(dev.index)))
    return (out, lse) if return_lse else out
