"""Attention over the paged cache against softmax in 64 bits.

Tolerances follow from the roundings, with u = 2^-11 (float16) or 2^-8 (bfloat16)
for one rounding to 16 bits, o the exact output and A = sum p |v| / sum p its
absolute companion.  The output is rounded once: u |o|.  window_attention rounds
each weight once before the second product: at most u A more (and, in float16,
2^-25 |v| for each weight too small for a normal number).  decode_attention keeps
24 bits of a weight.  Sums in float32 over n keys of products of 16-bit values add
at most 2^-22 (|q| |k| scale + 4) n^(1/2) A here, taken as 1e-4 A (n <= 20000,
scores below 50).  The log-sum-exp is float32: 1e-5 of its size plus 1e-5."""
import math

import numpy as np
import pytest
import torch

from quipsharp_b200 import _native as N
from quipsharp_b200 import attention as at
from quipsharp_b200 import kv_cache as kc

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make(rs, lengths, kv_heads, page, dim, dtype, width=None, spare=3, junk=0.0):
    """Pools and tables for the given lengths; everything that no row holds is `junk`."""
    lengths = np.asarray(lengths, np.int32)
    width = width or max(1, -(-int(lengths.max(initial=0)) // page))
    pages = int((-(-lengths // page)).sum()) + spare
    order = iter(rs.permutation(pages))
    table = np.full((len(lengths), width), -1, np.int32)
    g = torch.Generator(device=DEV).manual_seed(int(rs.randint(1 << 30)))
    k, v = (torch.randn(pages, kv_heads, page, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
    held = torch.zeros(pages, page, dtype=torch.bool, device=DEV)
    for i, n in enumerate(lengths):
        for c in range(-(-int(n) // page)):
            table[i, c] = next(order)
            held[int(table[i, c]), :min(page, int(n) - c * page)] = True
    for x in (k, v):
        x.masked_fill_(~held[:, None, :, None], junk)
    return k, v, torch.from_numpy(table).to(DEV), torch.from_numpy(lengths).to(DEV)


def exact(q, k, v, table, lengths, new, window, sinks, scale=None, hidden=()):
    """(out, lse, A) in 64 bits: row r's last new[r] tokens, packed; nobody sees the keys of
    the columns `hidden`."""
    page, dim = k.shape[2], k.shape[3]
    share = q.shape[1] // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    outs, lses, absolute, i = [], [], [], 0
    for r, t in enumerate(new):
        n = int(lengths[r])
        ids = table[r, :-(-n // page)].long()
        kk = k[ids].transpose(1, 2).reshape(-1, k.shape[1], dim)[:n].double().repeat_interleave(share, 1)
        vv = v[ids].transpose(1, 2).reshape(-1, k.shape[1], dim)[:n].double().repeat_interleave(share, 1)
        qq = q[i:i + t].double()
        i += t
        pos = n - t + torch.arange(t, device=DEV)[:, None]
        key = torch.arange(n, device=DEV)[None]
        see = key <= pos
        if window:
            see &= (key > pos - window) | (key < sinks)
        for c in hidden:
            see &= key // page != c
        s = torch.einsum("thd,nhd->htn", qq, kk) * scale
        s = s.masked_fill(~see, -math.inf)
        lse = torch.logsumexp(s, -1)
        p = torch.where(see, (s - torch.where(lse == -math.inf, 0.0, lse)[..., None]).exp(), 0.0)
        outs.append(torch.einsum("htn,nhd->thd", p, vv))
        absolute.append(torch.einsum("htn,nhd->thd", p, vv.abs()))
        lses.append(lse.T)
    return torch.cat(outs), torch.cat(lses), torch.cat(absolute)


def check(got, want, dtype, weights):
    out, lse = got
    o, l, a = want
    u = U[dtype]
    tol = u * o.abs() + 1e-4 * a + (u * a + 20000 * 2.0 ** -25 * 6 if weights else 0) + 1e-7
    err = (out.double() - o).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    assert torch.equal(torch.isneginf(lse), torch.isneginf(l))
    fin = torch.isfinite(l)
    assert bool(((lse.double() - l).abs() <= 1e-5 + 1e-5 * l.abs())[fin].all())


DECODE = [
    # lengths, q_heads, kv_heads, page, dim, window, sinks
    ([1], 1, 1, 16, 64, 0, 0),
    ([0, 1, 15, 16, 17, 0], 8, 2, 16, 64, 0, 0),
    ([203], 32, 8, 16, 128, 0, 0),
    ([33, 500, 1], 7, 1, 32, 80, 0, 0),
    ([64, 63, 65, 129], 24, 2, 64, 96, 0, 0),             # 12 heads share a key head
    ([100, 300], 40, 1, 16, 128, 0, 0),                   # 40 share one: three blocks of rows
    ([700, 40, 256, 257, 5], 4, 4, 256, 8, 0, 0),
    ([5000, 1, 900, 17, 0, 1024], 28, 4, 32, 64, 1000, 4),
    ([100, 90, 80, 20, 5], 8, 8, 16, 128, 30, 20),        # sinks and window share groups, or cover everything
    ([400, 401, 7], 2, 1, 128, 40, 1, 0),                 # a window of one token
    ([400, 401, 7], 2, 1, 128, 40, 3, 1000),              # all keys are sinks
    ([20000, 130, 11000], 16, 2, 64, 128, 0, 0),          # ranges shared by several CTAs
    ([9000] * 3 + [3] * 50, 8, 2, 16, 128, 0, 0),
    ([50 + 7 * i for i in range(200)], 4, 4, 16, 64, 0, 0),  # more rows than threads
    ([1100, 3, 0, 64, 1090], 8, 2, 16, 64, 0, 0),            # eight CTAs share a segment, some with nothing
    ([550, 1, 0, 300, 512, 20, 77, 490], 16, 8, 32, 128, 0, 0),  # four
    ([1500, 20, 3700], 48, 2, 64, 96, 0, 0),                 # two blocks of rows a key head
    ([3000, 4000, 10], 14, 2, 32, 64, 1100, 40),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths,q_heads,kv_heads,page,dim,window,sinks", DECODE)
def test_decode(lengths, q_heads, kv_heads, page, dim, window, sinks, dtype):
    rs = np.random.RandomState(len(lengths) + dim)
    k, v, table, n = make(rs, lengths, kv_heads, page, dim, dtype, junk=float("nan"))
    q = torch.randn(len(lengths), q_heads, dim, device=DEV).to(dtype)
    got = at.decode_attention(q, k, v, table, n, window=window or None, sinks=sinks, return_lse=True)
    check(got, exact(q, k, v, table, n, [1 if x else 0 for x in lengths], window, sinks) if min(lengths) else
          pad_empty(lengths, exact(q[torch.tensor(lengths, device=DEV) > 0], k, v, table, n, [1 if x else 0 for x in lengths],
                                   window, sinks)), dtype, weights=False)
    assert torch.equal(at.decode_attention(q, k, v, table, n, window=window or None, sinks=sinks), got[0])


def pad_empty(lengths, want):
    """Rows of length 0 in their places: zero outputs, lse -inf."""
    live = torch.tensor(lengths, device=DEV) > 0
    full = []
    for x, fill in zip(want, (0.0, -math.inf, 0.0)):
        y = torch.full((len(lengths), *x.shape[1:]), fill, device=DEV, dtype=torch.float64)
        y[live] = x
        full.append(y)
    return full


def test_decode_of_unseen_keys_whatever_they_hold():
    """NaN and infinities outside the window, and in pages that no row holds, do not enter."""
    rs = np.random.RandomState(1)
    k, v, table, n = make(rs, [300, 40], 2, 16, 64, torch.float16, junk=float("inf"))
    q = torch.randn(2, 4, 64, device=DEV).half()
    want = exact(q, k, v, table, n, [1, 1], 50, 5)
    for x in (k, v):
        for place in range(5, 250):
            x[int(table[0, place // 16]), :, place % 16] = float("nan")
    check(at.decode_attention(q, k, v, table, n, window=50, sinks=5, return_lse=True), want, torch.float16, False)


def test_nan_that_is_seen_shows():
    rs = np.random.RandomState(2)
    k, v, table, n = make(rs, [40, 20], 1, 16, 64, torch.float16)
    q = torch.randn(2, 2, 64, device=DEV).half()
    q[1] = float("nan")
    k[int(table[0, 1]), 0, 3, 5] = float("nan")
    out, lse = at.decode_attention(q, k, v, table, n, return_lse=True)
    assert out.isnan().all() and lse.isnan().all()
    out, lse = at.window_attention(q, k, v, table, n, torch.tensor([0, 1, 2], device=DEV, dtype=torch.int32), return_lse=True)
    assert out.isnan().all() and lse.isnan().all()


def test_absent_pages_and_overlong_rows():
    """Entries of -1, or beyond the pool, are keys that do not exist; a length beyond the line ends with it."""
    rs = np.random.RandomState(3)
    k, v, table, n = make(rs, [160, 160], 2, 16, 64, torch.bfloat16)
    q = torch.randn(2, 4, 64, device=DEV).bfloat16()
    whole = table.clone()
    gone = torch.arange(160, device=DEV)
    gone = (gone // 16 == 2) | (gone // 16 == 9)
    table[0, 2], table[0, 9] = -1, 1 << 20
    kz = k.clone()
    big = exact(q, kz, v, whole, n, [1, 1], 0, 0)
    # the same keys hidden: a cache without them, in the same order
    keep = torch.tensor([c for c in range(10) if c not in (2, 9)], device=DEV)
    sub = exact(q[:1], k, v, whole[:1, keep], torch.tensor([128]), [1], 0, 0)
    want = [torch.cat([s, b[1:]]) for s, b in zip(sub, big)]
    check(at.decode_attention(q, k, v, table, n, return_lse=True), want, torch.bfloat16, False)
    cu = torch.tensor([0, 1, 2], device=DEV, dtype=torch.int32)
    check(at.window_attention(q, k, v, table, n, cu, return_lse=True), want, torch.bfloat16, True)
    long = n + 500
    got = at.decode_attention(q, k, v, whole, long, return_lse=True)
    check(got, big, torch.bfloat16, False)


def test_strided_queries_and_token_major_pools():
    rs = np.random.RandomState(4)
    k, v, table, n = make(rs, [77, 300, 16], 4, 32, 64, torch.float16)
    kt, vt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    joint = torch.randn(3, 8 + 4 + 4, 64, device=DEV).half()
    q = joint[:, :8]
    want = exact(q, k, v, table, n, [1, 1, 1], 0, 0)
    check(at.decode_attention(q, kt, vt, table, n, return_lse=True), want, torch.float16, False)
    cu = torch.arange(4, device=DEV, dtype=torch.int32)
    check(at.window_attention(q, kt, vt, table, n, cu, return_lse=True), want, torch.float16, True)
    odd = torch.randn(3, 8, 72, device=DEV).half()[..., 4:68]  # an unaligned start: copied
    check(at.decode_attention(odd, k, v, table, n, return_lse=True), exact(odd, k, v, table, n, [1, 1, 1], 0, 0),
          torch.float16, False)


def test_scale_and_large_scores():
    rs = np.random.RandomState(5)
    k, v, table, n = make(rs, [500, 129], 1, 16, 128, torch.float16)
    k[:, :, :, 0] *= 20  # a channel that dominates: scores up to about +-50, maxima that keep growing
    q = torch.randn(2, 4, 128, device=DEV).half()
    q[:, :, 0] = 2.0
    cu = torch.tensor([0, 1, 2], device=DEV, dtype=torch.int32)
    for scale in (0.3, 1.0):
        want = exact(q, k, v, table, n, [1, 1], 0, 0, scale)
        check(at.decode_attention(q, k, v, table, n, scale=scale, return_lse=True), want, torch.float16, False)
        check(at.window_attention(q, k, v, table, n, cu, scale=scale, return_lse=True), want, torch.float16, True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_first_token_that_takes_the_weight_and_has_no_value(dtype):
    """The others' weights, 2^-20 of the first one's, decide the output: none may fall out of
    float16's normal range, so the roundings are those of the other tests without an
    absolute part."""
    rs = np.random.RandomState(10)
    n = 600
    k, v, table, lengths = make(rs, [n], 1, 16, 64, dtype)
    q = torch.randn(3, 4, 64, device=DEV).to(dtype)
    q[:, :, 0] = 4.0
    k[:, :, :, 0] = 0
    v *= 200
    first = int(table[0, 0])
    k[first, 0, 0], v[first, 0, 0] = 0, 0
    k[first, 0, 0, 0] = 28.0  # a score of 4 * 28 / 8 = 14 above the others' mean
    cu = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    for got, new, u in ((at.window_attention(q, k, v, table, lengths, cu), 3, 2 * U[dtype]),
                        (at.decode_attention(q[2:], k, v, table, lengths), 1, U[dtype])):
        o, _, a = exact(q[3 - new:], k, v, table, lengths, [new], 0, 0)
        assert float(a.max()) < 1.0
        err = (got.double() - o).abs()
        assert bool((err <= u * (o.abs() + a) + 1e-4 * a + 2.0 ** -25).all()), float((err / a).max())


def test_pools_past_32_bit_offsets():
    """A pool of more than 2^32 bytes, with the row's pages at its end."""
    pages = (1 << 31) // (2 * 64 * 64) + 40
    k = torch.zeros(pages, 2, 64, 64, dtype=torch.float16, device=DEV)
    v = torch.zeros_like(k)
    rs = np.random.RandomState(6)
    sk, sv, _, n = make(rs, [150], 2, 64, 64, torch.float16, spare=0)
    k[-3:], v[-3:] = sk, sv
    table = torch.tensor([[pages - 2, pages - 1, pages - 3]], dtype=torch.int32, device=DEV)
    q = torch.randn(1, 4, 64, device=DEV).half()
    want = exact(q, k, v, table, n, [1], 0, 0)
    check(at.decode_attention(q, k, v, table, n, return_lse=True), want, torch.float16, False)
    check(at.window_attention(q, k, v, table, n, torch.tensor([0, 1], device=DEV, dtype=torch.int32), return_lse=True), want,
          torch.float16, True)


WINDOW = [
    # new, past, q_heads, kv_heads, page, dim, window, sinks
    ([1], [0], 1, 1, 16, 64, 0, 0),
    ([5, 0, 1, 17], [3, 9, 0, 100], 4, 2, 16, 64, 0, 0),
    ([128], [0], 2, 2, 16, 128, 0, 0),
    ([129, 127], [1, 130], 8, 2, 32, 128, 0, 0),
    ([300, 40], [0, 77], 8, 1, 64, 96, 0, 0),
    ([200], [300], 14, 2, 128, 80, 0, 0),                  # 7 heads share: 18 tokens of 128 rows
    ([70], [500], 128, 1, 256, 64, 0, 0),                  # 128 heads share: one token a tile
    ([33, 600], [600, 0], 6, 3, 16, 40, 0, 0),
    ([600, 90], [0, 800], 8, 2, 16, 128, 100, 4),
    ([600, 90], [0, 800], 8, 2, 256, 64, 100, 150),        # sinks reach past a key tile
    ([500], [20], 16, 2, 64, 128, 1, 0),                   # each token sees itself
    ([500], [20], 16, 2, 64, 128, 7, 700),                 # all keys are sinks
    ([1000], [3000], 4, 1, 128, 128, 1024, 130),
    ([9, 1, 4], [700, 30, 250], 16, 4, 16, 64, 256, 4),
    ([2, 3, 1] * 40, [10, 50, 300] * 40, 8, 2, 16, 64, 64, 2),  # more rows than a warp
    ([1500], [0], 8, 8, 64, 128, 0, 0),
    ([8], [15000], 8, 1, 64, 128, 0, 0),                   # few tokens over many keys: shares of the keys, joined
    ([5, 0, 70, 1], [9000, 50, 40, 0], 8, 2, 32, 64, 0, 0),   # shares that are empty for the short rows
    ([3, 2], [15000, 2000], 6, 2, 16, 96, 5000, 300),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,past,q_heads,kv_heads,page,dim,window,sinks", WINDOW)
def test_window(new, past, q_heads, kv_heads, page, dim, window, sinks, dtype):
    rs = np.random.RandomState(sum(new) + dim)
    k, v, table, n = make(rs, [a + b for a, b in zip(new, past)], kv_heads, page, dim, dtype, junk=float("nan"))
    q = torch.randn(sum(new), q_heads, dim, device=DEV).to(dtype)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]).astype(np.int32), device=DEV)
    got = at.window_attention(q, k, v, table, n, cu, window=window or None, sinks=sinks, return_lse=True)
    check(got, exact(q, k, v, table, n, new, window, sinks), dtype, weights=True)
    assert torch.equal(at.window_attention(q, k, v, table, n, cu, window=window or None, sinks=sinks), got[0])
    assert N.lib().qs_device_status(N.stream_of(q)) == N.QS_OK


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (128, 128)])
@pytest.mark.parametrize("hidden", [(), (3, 4)])
def test_edges_at_every_place_of_a_key_tile(dim, page, hidden):
    """Windows, sinks and starts that put the edges of what a query tile sees before, at and
    after each 32 keys of a tile, with pages missing too."""
    rs = np.random.RandomState(dim + page)
    new, past = [150, 33, 1], [130, 421, 255]
    k, v, table, n = make(rs, [a + b for a, b in zip(new, past)], 2, page, dim, torch.float16)
    q = torch.randn(sum(new), 16, dim, device=DEV).half()
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]).astype(np.int32), device=DEV)
    lines = table.clone()
    for c in hidden:
        if c < table.shape[1]:
            table[:, c] = -1
    for window in (1, 2, 31, 32, 33, 63, 64, 65, 95, 97, 127, 128, 129, 161, 200, 300):
        for sinks in (0, 1, 33, 65, 100, 129):
            got = at.window_attention(q, k, v, table, n, cu, window=window, sinks=sinks, return_lse=True)
            check(got, exact(q, k, v, lines, n, new, window, sinks, hidden=hidden), torch.float16, weights=True)


def test_window_tokens_of_no_row_are_zero():
    rs = np.random.RandomState(7)
    k, v, table, n = make(rs, [50, 20], 2, 16, 64, torch.float16)
    q = torch.randn(400, 8, 64, device=DEV).half()
    cu = torch.tensor([0, 30, 45], device=DEV, dtype=torch.int32)
    out, lse = at.window_attention(q, k, v, table, n, cu, return_lse=True)
    check((out[:45], lse[:45]), exact(q, k, v, table, n, [30, 15], 0, 0), torch.float16, True)
    assert not out[45:].any() and torch.isneginf(lse[45:]).all()


def test_decode_is_window_of_one():
    rs = np.random.RandomState(8)
    k, v, table, n = make(rs, [500, 3, 77], 2, 16, 128, torch.bfloat16)
    q = torch.randn(3, 8, 128, device=DEV).bfloat16()
    a = at.decode_attention(q, k, v, table, n, window=60, sinks=4).float()
    b = at.window_attention(q, k, v, table, n, torch.arange(4, device=DEV, dtype=torch.int32), window=60, sinks=4).float()
    assert float((a - b).norm() / a.norm()) < 2 ** -7


def test_repeats_exactly_on_any_stream_and_in_a_graph():
    rs = np.random.RandomState(9)
    k, v, table, n = make(rs, [3000, 10, 700], 2, 16, 64, torch.float16)
    q = torch.randn(3, 8, 64, device=DEV).half()
    cu = torch.arange(4, device=DEV, dtype=torch.int32)
    want = [at.decode_attention(q, k, v, table, n), at.window_attention(q, k, v, table, n, cu)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [at.decode_attention(q, k, v, table, n), at.window_attention(q, k, v, table, n, cu)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [at.decode_attention(q, k, v, table, n), at.window_attention(q, k, v, table, n, cu)]
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_empty_calls():
    k = torch.zeros(4, 2, 16, 64, device=DEV, dtype=torch.float16)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    q = torch.zeros(0, 4, 64, device=DEV, dtype=torch.float16)
    assert at.decode_attention(q, k, k, torch.zeros(0, 3, dtype=torch.int32, device=DEV), none).shape == (0, 4, 64)
    table, n = torch.zeros(2, 3, dtype=torch.int32, device=DEV), torch.tensor([5, 6], dtype=torch.int32, device=DEV)
    assert at.window_attention(q, k, k, table, n, torch.zeros(3, dtype=torch.int32, device=DEV)).shape == (0, 4, 64)
    empty = torch.zeros(2, 0, dtype=torch.int32, device=DEV)  # lines without a page
    out = at.decode_attention(torch.ones(2, 4, 64, device=DEV).half(), k, k, empty, n)
    assert not out.any()


def test_arguments_that_need_a_copy_or_a_refusal():
    """What the direct call does not take goes the longer way and gives the same, or its error."""
    rs = np.random.RandomState(11)
    k, v, table, n = make(rs, [77, 300, 16], 4, 32, 64, torch.float16)
    q = torch.randn(3, 8, 64, device=DEV).half()
    cu = torch.arange(4, device=DEV, dtype=torch.int32)
    decode = at.decode_attention(q, k, v, table, n)
    window = at.window_attention(q, k, v, table, n, cu)
    wide = torch.stack((table, table), -1)[..., 0]
    twice = torch.stack((n, n), -1)[:, 0]
    unaligned = torch.empty(3 * 8 * 64 + 1, device=DEV, dtype=torch.float16)[1:].view(3, 8, 64).copy_(q)
    assert not wide.is_contiguous() and not twice.is_contiguous() and unaligned.data_ptr() % 16
    for args in ((q, k, v, wide, n), (q, k, v, table, twice), (unaligned, k, v, table, n)):
        assert torch.equal(at.decode_attention(*args), decode)
        assert torch.equal(at.window_attention(*args, cu), window)
    assert torch.equal(at.decode_attention(q, k, v, table, n, window=np.int64(1000), scale=np.float64(0.125)), decode)
    grad = q.clone().requires_grad_()
    for error, call in (
            (TypeError, lambda: at.decode_attention(q.bfloat16(), k, v, table, n)),
            (TypeError, lambda: at.decode_attention(q, k, v, table.long(), n)),
            (TypeError, lambda: at.window_attention(q, k, v, table, n, cu.long())),
            (ValueError, lambda: at.decode_attention(q[:2], k, v, table, n)),
            (ValueError, lambda: at.decode_attention(q, k, v, table, n, window=0)),
            (ValueError, lambda: at.window_attention(q, k, v, table, n, cu[:3])),
            (RuntimeError, lambda: at.decode_attention(grad, k, v, table, n)),
            (RuntimeError, lambda: at.decode_attention(q, k, v, table.cpu(), n)),
            (RuntimeError, lambda: at.decode_attention(q, k, v, table, n, scale=-1.0)),
            (NotImplementedError, lambda: at.decode_attention(q, k[:, :, :24], v[:, :, :24], table, n))):
        with pytest.raises(error):
            call()
    with torch.no_grad():
        assert torch.equal(at.decode_attention(grad, k, v, table, n), decode)
