"""A paged key-value cache for decoding with quantized layers.

The reference leaves decoding to transformers; this module and `attention` are
what a decoder of QuantizedLinear layers needs beside its products.  A cache
keeps the keys and values of every layer in pages of `page_size` tokens; a row
(one sequence, or one beam of a search) is a line of page numbers in `table`
with its length in tokens, and `refcount` holds how many references each page
has.  All bookkeeping runs on the device, without a synchronisation, and a page
is taken by a fixed rule (the lowest free one), so results repeat exactly.

* `PagedKVCache` keeps the state and updates it in place (its tensors stay
  where they are, so its calls can be captured in CUDA graphs).
* `fork_pages`, `compact_pages`, `extend_pages` and `write_kv` are the same
  operations on tensors that the caller keeps.  The tables and counts come back
  as new tensors; the pools are changed in place.

What the kernels find wrong on the device (no free page left, a parent out of
range) never stops a stream: `check_device()` synchronises and raises it.
"""
from __future__ import annotations

import torch
from torch import Tensor

from . import _native as N

KV_DTYPES = {torch.float16: N.QS_F16, torch.bfloat16: N.QS_BF16}


def check_device(device=None) -> None:
    """Synchronises the current stream and raises what the kernels found wrong
    since the last call, on any cache of the device: RuntimeError when rows found
    no free page or a bounded wait ran out, IndexError for a parent or token count
    out of range.  One kind at a time: where there are two, the next call raises
    the other."""
    with torch.cuda.device(device):
        N.check(N.lib().qs_device_status(N.raw_stream(torch.cuda.current_device())))


def _int32(name: str, t: Tensor, *shape) -> Tensor:
    if t.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _device_of(first: Tensor, *others) -> int:
    """The index of the one CUDA device that holds all the tensors."""
    index = first.get_device()
    if index < 0:
        N.require_cuda(first)
    for t in others:
        if t is not None and t.get_device() != index:
            N.require_cuda(t)
            raise ValueError(f"all tensors must be on one device, got {first.device} and {t.device}")
    return index


def kv_pool(k: Tensor, v: Tensor):
    """(description for the library, pages, heads, page, dim) of pools k, v
    (layers, pages, heads, page, dim) or, of one layer, (pages, heads, page, dim)."""
    dtype = KV_DTYPES.get(k.dtype)
    if dtype is None or v.dtype is not k.dtype:
        raise TypeError(f"a cache holds float16 or bfloat16 keys and values of one type, got {k.dtype} and {v.dtype}")
    shape, ks, vs = k.shape, k.stride(), v.stride()
    if v.shape != shape or len(shape) not in (4, 5):
        raise ValueError("key and value pools must have one shape, ([layers,] pages, heads, page, dim); "
                         f"got {tuple(k.shape)} and {tuple(v.shape)}")
    if ks[-1] != 1 or vs[-1] != 1:
        raise ValueError("the last dimension of a pool must be contiguous")
    if len(shape) == 4:
        shape, ks, vs = (1, *shape), (0, *ks), (0, *vs)
    return (N.pack_kv_pool(k.data_ptr(), v.data_ptr(), dtype, *shape, *ks[:4], *vs[:4]), *shape[1:])


def _workspace(rows: int, pages: int, like: Tensor) -> tuple[Tensor, int]:
    n = N.workspace_bytes("qs_cache_workspace_bytes", rows, pages)
    if n < 0:
        raise NotImplementedError(f"a cache has 1 to 2^28 pages and at most 8192 rows, got {pages} pages, {rows} rows")
    return like.new_empty(n // 4), n


def _state(k: Tensor, v: Tensor, table: Tensor, lengths: Tensor, refcount: Tensor):
    if table.dim() != 2:
        raise ValueError(f"table must be (rows, width), got {tuple(table.shape)}")
    rows, width = table.shape
    pool, pages = kv_pool(k, v)[:2]
    return (pool, pages, rows, width, _int32("table", table, rows, width), _int32("lengths", lengths, rows),
            _int32("refcount", refcount, pages))


def fork_pages(k: Tensor, v: Tensor, table: Tensor, lengths: Tensor, refcount: Tensor,
               parents: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """Every row i becomes a copy of row parents[i] (-1: empty): fork, free and
    reorder at once.

    Whole pages are shared; a part-filled last page stays with a row's lowest
    child, and each other child gets the lowest free page with the filled tokens
    of all layers copied.  Returns the new (table, lengths, refcount); the pools
    k, v (layers, pages, heads, page, dim) are changed in place.  refcount may
    hold references of the caller's besides the table's: they stay."""
    got = N.fast().fork_pages(k, v, table, lengths, refcount, parents)
    if got is not None:
        return got
    N.refuse_grad("fork_pages", k, v)
    dev = _device_of(k, v, table, lengths, refcount, parents)
    if not N.is_current(dev):
        with torch.cuda.device(dev):
            return fork_pages(k, v, table, lengths, refcount, parents)
    pool, pages, rows, width, table, lengths, refcount = _state(k, v, table, lengths, refcount)
    parents = _int32("parents", parents, rows)
    ws, nb = _workspace(rows, pages, table)
    t, n, c = torch.empty_like(table), torch.empty_like(lengths), torch.empty_like(refcount)
    N.check(N.lib().qs_cache_fork(pool, rows, width, table.data_ptr(), lengths.data_ptr(), refcount.data_ptr(),
                                  parents.data_ptr(), t.data_ptr(), n.data_ptr(), c.data_ptr(), ws.data_ptr(), nb,
                                  N.raw_stream(dev)))
    return t, n, c


def compact_pages(k: Tensor, v: Tensor, table: Tensor, lengths: Tensor,
                  refcount: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    """Moves the pages in use to the lowest page numbers: with U of them, those
    from U on go to the holes below U, both in ascending order.  Returns the new
    (table, refcount, U as an int32 tensor of one); the pools are changed in
    place, and pages from U on are free."""
    got = N.fast().compact_pages(k, v, table, lengths, refcount)
    if got is not None:
        return got
    N.refuse_grad("compact_pages", k, v)
    dev = _device_of(k, v, table, lengths, refcount)
    if not N.is_current(dev):
        with torch.cuda.device(dev):
            return compact_pages(k, v, table, lengths, refcount)
    pool, pages, rows, width, table, lengths, refcount = _state(k, v, table, lengths, refcount)
    ws, nb = _workspace(rows, pages, table)
    t, c, used = torch.empty_like(table), torch.empty_like(refcount), refcount.new_empty(1)
    N.check(N.lib().qs_cache_compact(pool, rows, width, table.data_ptr(), lengths.data_ptr(), refcount.data_ptr(),
                                     t.data_ptr(), c.data_ptr(), used.data_ptr(), ws.data_ptr(), nb, N.raw_stream(dev)))
    return t, c, used


def extend_pages(table: Tensor, lengths: Tensor, refcount: Tensor, new_tokens: Tensor,
                 page_size: int) -> tuple[Tensor, Tensor, Tensor]:
    """Every row i grows by new_tokens[i] tokens; the pages that it needs are the
    lowest free ones, in row and then column order.  Returns the new (table,
    lengths, refcount).  A row that finds no page, or outgrows its line, has -1
    there: its tokens are left out, and `check_device` raises."""
    got = N.fast().extend_pages(table, lengths, refcount, new_tokens, page_size)
    if got is not None:
        return got
    dev = _device_of(table, lengths, refcount, new_tokens)
    if not N.is_current(dev):
        with torch.cuda.device(dev):
            return extend_pages(table, lengths, refcount, new_tokens, page_size)
    if table.dim() != 2 or refcount.dim() != 1:
        raise ValueError("table must be (rows, width) and refcount (pages,), "
                         f"got {tuple(table.shape)} and {tuple(refcount.shape)}")
    rows, width = table.shape
    table, lengths = _int32("table", table, rows, width), _int32("lengths", lengths, rows)
    refcount, new_tokens = _int32("refcount", refcount, len(refcount)), _int32("new_tokens", new_tokens, rows)
    t, n, c = torch.empty_like(table), torch.empty_like(lengths), torch.empty_like(refcount)
    _extend(page_size, table, lengths, refcount, new_tokens, t, n, c, dev)
    return t, n, c


def _extend(page_size, table, lengths, refcount, new_tokens, t, n, c, dev) -> None:
    rows, width = table.shape
    pages = len(refcount)
    ws, nb = _workspace(rows, pages, table)
    N.check(N.lib().qs_cache_extend(page_size, pages, rows, width, table.data_ptr(), lengths.data_ptr(),
                                    refcount.data_ptr(), new_tokens.data_ptr(), t.data_ptr(), n.data_ptr(),
                                    c.data_ptr(), ws.data_ptr(), nb, N.raw_stream(dev)))


def write_kv(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor,
             cu: Tensor | None = None) -> None:
    """Writes new tokens' keys and values k, v (tokens, heads, dim) into one
    layer's pools (pages, heads, page, dim).  Row r's tokens are [cu[r],
    cu[r+1]) and take its last places, which `lengths` already counts; without
    cu every row has one.  k and v may be views (the last dimension
    contiguous)."""
    if N.fast().write_kv(k, v, k_pages, v_pages, table, lengths, cu):
        return
    N.refuse_grad("write_kv", k, v, k_pages, v_pages)
    dev = _device_of(k, v, k_pages, v_pages, table, lengths, cu)
    if not N.is_current(dev):
        with torch.cuda.device(dev):
            return write_kv(k, v, k_pages, v_pages, table, lengths, cu)
    if k_pages.dim() != 4 or table.dim() != 2:
        raise ValueError("write_kv takes one layer's pools (pages, heads, page, dim) and a table (rows, width)")
    pool, _, heads, _, dim = kv_pool(k_pages, v_pages)
    rows, width = table.shape
    table, lengths = _int32("table", table, rows, width), _int32("lengths", lengths, rows)
    if cu is not None:
        cu = _int32("cu", cu, rows + 1)
    if k.dtype is not k_pages.dtype or v.dtype is not k_pages.dtype:
        raise TypeError(f"keys and values must have the pools' type {k_pages.dtype}, got {k.dtype} and {v.dtype}")
    shape = k.shape
    if len(shape) != 3 or v.shape != shape or shape[1] != heads or shape[2] != dim:
        raise ValueError(f"keys and values must be (tokens, {heads}, {dim}), got {tuple(k.shape)} and {tuple(v.shape)}")
    k, v = N.rows_of_8(k), N.rows_of_8(v)
    ks, vs = k.stride(), v.stride()
    N.check(N.lib().qs_cache_write(pool, rows, width, table.data_ptr(), lengths.data_ptr(),
                                   None if cu is None else cu.data_ptr(), k.data_ptr(), ks[0], ks[1], v.data_ptr(),
                                   vs[0], vs[1], shape[0], N.raw_stream(dev)))


class PagedKVCache:
    """The keys and values of `layers` layers for up to `rows` sequences of up to
    `max_len` tokens, in `num_pages` pages of `page_size` tokens.

    A decoding step: `extend(new)` takes pages for the rows' new tokens, then
    each layer writes its keys and values (`write`) and reads them (`decode`,
    `window`).  `fork(parents)` shares, reorders and frees rows.  The state
    (`k`, `v`, `table`, `lengths`, `refcount`) is updated in place."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, num_pages: int, rows: int, max_len: int,
                 page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if dtype not in KV_DTYPES:
            raise TypeError(f"a cache holds float16 or bfloat16, got {dtype}")
        if min(layers, kv_heads, num_pages, rows, max_len) < 1:
            raise ValueError("layers, kv_heads, num_pages, rows and max_len must be positive")
        if page_size not in (16, 32, 64, 128, 256):
            raise NotImplementedError(f"page size must be a power of two of 16 to 256, got {page_size}")
        if head_dim % 8 or not 0 < head_dim <= 128:
            raise NotImplementedError(f"head dimension must be a multiple of 8 up to 128, got {head_dim}")
        shape = (layers, num_pages, kv_heads, page_size, head_dim)
        self.page_size, self.max_len = page_size, max_len
        self.k, self.v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        N.require_cuda(self.k)
        device = self.k.device
        self.table = torch.full((rows, -(-max_len // page_size)), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=device)
        self.refcount = torch.zeros(num_pages, dtype=torch.int32, device=device)

    def extend(self, new_tokens) -> None:
        """Every row i grows by new_tokens[i] (an int32 tensor, or one number for
        all rows)."""
        if not isinstance(new_tokens, Tensor):
            new_tokens = torch.full_like(self.lengths, int(new_tokens))
        dev = _device_of(self.table, new_tokens)
        new_tokens = _int32("new_tokens", new_tokens, len(self.lengths))
        with torch.cuda.device(dev):
            _extend(self.page_size, self.table, self.lengths, self.refcount, new_tokens, self.table, self.lengths,
                    self.refcount, dev)

    def write(self, layer: int, k: Tensor, v: Tensor, cu: Tensor | None = None) -> None:
        """New tokens' keys and values of one layer (see write_kv)."""
        write_kv(k, v, self.k[layer], self.v[layer], self.table, self.lengths, cu)

    def decode(self, layer: int, q: Tensor, **options) -> Tensor:
        """attention.decode_attention of the rows' newest tokens."""
        from .attention import decode_attention
        return decode_attention(q, self.k[layer], self.v[layer], self.table, self.lengths, **options)

    def window(self, layer: int, q: Tensor, cu: Tensor, **options) -> Tensor:
        """attention.window_attention of the rows' new tokens."""
        from .attention import window_attention
        return window_attention(q, self.k[layer], self.v[layer], self.table, self.lengths, cu, **options)

    def fork(self, parents: Tensor) -> None:
        """Every row i becomes a copy of row parents[i], -1: empty (see fork_pages)."""
        t, n, c = fork_pages(self.k, self.v, self.table, self.lengths, self.refcount, parents)
        self.table.copy_(t)
        self.lengths.copy_(n)
        self.refcount.copy_(c)

    def free(self, rows) -> None:
        """Empties the given rows (a list of numbers, or a boolean or index tensor)."""
        parents = torch.arange(self.lengths.shape[0], dtype=torch.int32, device=self.lengths.device)
        parents[rows if isinstance(rows, Tensor) else list(rows)] = -1
        self.fork(parents)

    def compact(self) -> Tensor:
        """Moves the pages in use together; returns their number (int32 tensor of one)."""
        t, c, used = compact_pages(self.k, self.v, self.table, self.lengths, self.refcount)
        self.table.copy_(t)
        self.refcount.copy_(c)
        return used

    def check(self) -> None:
        """Raises what the kernels found wrong since the last check, on any cache of
        the device (see check_device)."""
        check_device(self.k.device)
