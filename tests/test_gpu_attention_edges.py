"""Attention over the paged cache at the edges of what a row, a table and a pool may hold
(see test_gpu_attention for the exact form and the tolerances)."""
import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwd

from quipsharp_b200 import _native as N
from quipsharp_b200 import attention as at
from quipsharp_b200 import kv_cache as kc
from quipsharp_b200.beam import beam_select
from test_gpu_attention import DEV, check, exact, make

pytestmark = pytest.mark.gpu


def offsets(new, first=0):
    return torch.tensor(np.concatenate([[0], np.cumsum(new)]) + first, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,page,width,dim,window,sinks", [
    ([1, 1], 16, 10, 64, 0, 0), ([9, 40], 16, 10, 128, 0, 0), ([9, 40], 16, 10, 64, 600, 0), ([5, 300], 32, 7, 80, 40, 500),
    ([5, 3], 16, 201, 64, 0, 0), ([3, 200], 16, 11, 64, 30, 0), ([20, 7], 64, 3, 128, 600, 130)])
def test_rows_that_outgrew_their_line(new, page, width, dim, window, sinks, dtype):
    """A length past width x page: its keys end with the line, whatever place a token has."""
    rs = np.random.RandomState(width)
    held = width * page
    k, v, table, n = make(rs, [held, held], 2, page, dim, dtype)
    q = torch.randn(sum(new), 8, dim, device=DEV).to(dtype)
    # what an earlier call left in shared memory is large
    big = torch.full((2, held, 2, dim), 30.0, device=DEV, dtype=dtype).view(2 * width, page, 2, dim).transpose(1, 2).contiguous()
    lines = torch.arange(2 * width, dtype=torch.int32, device=DEV).view(2, width)
    for past in (0, 1, 13, 500):
        at.window_attention(q, big, big, lines, n, offsets(new))
        lengths = n + past
        got = at.window_attention(q, k, v, table, lengths, offsets(new), window=window or None, sinks=sinks, return_lse=True)
        check(got, bounded(q, k, v, table, lengths.tolist(), held, new, window, sinks), dtype, weights=True)
        last = torch.tensor(np.cumsum(new) - 1, device=DEV)
        one = at.decode_attention(q[last], k, v, table, lengths, window=window or None, sinks=sinks, return_lse=True)
        want = bounded(q[last], k, v, table, lengths.tolist(), held, [1, 1], window, sinks)
        check(one, want, dtype, weights=False)


def bounded(q, k, v, table, lengths, held, new, window, sinks):
    """exact for rows of any length, whose keys end at `held`."""
    parts, i = [], 0
    share, dim = q.shape[1] // k.shape[1], q.shape[2]
    for r, t in enumerate(new):
        kk, vv = (x[table[r].long()].transpose(1, 2).reshape(held, -1, dim).double().repeat_interleave(share, 1) for x in (k, v))
        pos = lengths[r] - t + torch.arange(t, device=DEV)[:, None]
        key = torch.arange(held, device=DEV)[None]
        see = key <= pos
        if window:
            see &= (key > pos - window) | (key < sinks)
        s = torch.einsum("thd,nhd->htn", q[i:i + t].double(), kk) * dim ** -0.5
        s = s.masked_fill(~see, -torch.inf)
        lse = torch.logsumexp(s, -1)
        p = torch.where(see, (s - torch.where(lse == -torch.inf, 0.0, lse)[..., None]).exp(), 0.0)
        parts.append((torch.einsum("htn,nhd->thd", p, vv), lse.T, torch.einsum("htn,nhd->thd", p, vv.abs())))
        i += t
    return [torch.cat(x) for x in zip(*parts)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,past,q_heads,kv_heads,page,dim,window,sinks,bad", [
    ([300, 40], [0, 77], 8, 2, 16, 64, 0, 0, [[0, 5, 130, 131, 299], [80, 116]]),   # seen by later tokens alone
    ([200], [300], 14, 2, 128, 80, 0, 0, [[310, 499]]),
    ([600, 9], [0, 800], 8, 1, 16, 128, 100, 4, [[4, 3, 250, 599], [2, 50, 650, 704, 805]]),  # before, after and between
    ([5], [5000], 4, 1, 64, 64, 100, 4, [[4, 50, 100, 4890, 4903]]),                # few tokens: shares of the keys
    ([3, 2], [9000, 40], 6, 2, 32, 96, 0, 0, [[9001, 9002], [41]]),
    ([130], [20], 128, 1, 32, 64, 33, 1, [[1, 60, 149]])])
def test_values_that_a_token_does_not_see_do_not_enter(new, past, q_heads, kv_heads, page, dim, window, sinks, bad, dtype):
    """NaN and infinite values of a key reach the tokens that see it, in their dimension,
    and no others: not those of the same tile either."""
    rs = np.random.RandomState(sum(new))
    k, v, table, n = make(rs, [a + b for a, b in zip(new, past)], kv_heads, page, dim, dtype, junk=float("nan"))
    q = torch.randn(sum(new), q_heads, dim, device=DEV).to(dtype)
    want = exact(q, k, v, table, n, new, window, sinks)
    hit = torch.zeros(sum(new), dim, dtype=torch.bool, device=DEV)
    start = 0
    for r, places in enumerate(bad):
        pos = past[r] + torch.arange(new[r], device=DEV)
        for i, place in enumerate(places):
            d = (7 * i + 3) % dim
            v[int(table[r, place // page]), :, place % page, d] = (float("nan"), float("inf"), -float("inf"))[i % 3]
            see = (place <= pos) & ((place > pos - window) | (place < sinks) if window else True)
            hit[start:start + new[r], d] |= see
        start += new[r]
    out, lse = at.window_attention(q, k, v, table, n, offsets(new), window=window or None, sinks=sinks, return_lse=True)
    hit = hit[:, None].expand(-1, q_heads, -1)
    assert not out[hit].isfinite().any()
    check((out.masked_fill(hit, 0), lse), (want[0].masked_fill(hit, 0), want[1], want[2]), dtype, weights=True)
    again = at.window_attention(q, k, v, table, n, offsets(new), window=window or None, sinks=sinks)
    assert torch.equal(again.masked_fill(hit, 0), out.masked_fill(hit, 0))


@pytest.mark.parametrize("first,new,past", [(1, [30, 15], [20, 5]), (300, [30, 15], [20, 5]), (45, [0, 200], [0, 7]),
                                            (5, [1], [3000])])
def test_tokens_before_the_first_row_are_zero(first, new, past):
    """cu[0] > 0, as of a slice of a larger batch: the tokens before it belong to no row."""
    rs = np.random.RandomState(first)
    k, v, table, n = make(rs, [a + b for a, b in zip(new, past)], 2, 16, 64, torch.float16)
    total = first + sum(new) + 33
    q = torch.randn(total, 8, 64, device=DEV).half()
    left = [torch.full(shape, float("nan"), device=DEV, dtype=t) for shape, t in
            (((total, 8, 64), torch.float16), ((total, 8), torch.float32))]  # what the outputs' memory held
    torch.cuda.synchronize()
    del left
    out, lse = at.window_attention(q, k, v, table, n, offsets(new, first), return_lse=True)
    mine = slice(first, first + sum(new))
    check((out[mine], lse[mine]), exact(q[mine], k, v, table, n, new, 0, 0), torch.float16, True)
    for rest in (slice(0, first), slice(first + sum(new), total)):
        assert not out[rest].any() and torch.isneginf(lse[rest]).all()


def test_pools_without_a_key_head_are_refused():
    k = torch.zeros(4, 0, 16, 64, device=DEV, dtype=torch.float16)
    q = torch.zeros(2, 4, 64, device=DEV, dtype=torch.float16)
    table, n = (torch.zeros(s, dtype=torch.int32, device=DEV) for s in ((2, 3), (2,)))
    for call in (lambda: at.decode_attention(q, k, k, table, n), lambda: at.window_attention(q, k, k, table, n, offsets([1, 1]))):
        with pytest.raises(ValueError, match="0 key heads"):
            call()


def test_pools_that_require_grad_are_refused():
    """No gradient reaches a pool: a call that would lose one is refused, as for the queries."""
    rs = np.random.RandomState(1)
    k, v, table, n = make(rs, [40, 20], 2, 16, 64, torch.float16)
    q = torch.randn(2, 4, 64, device=DEV).half()
    new = torch.randn(2, 2, 64, device=DEV).half()
    cu = torch.arange(3, dtype=torch.int32, device=DEV)
    count = torch.ones(len(k), dtype=torch.int32, device=DEV)
    grad = [x.clone().requires_grad_() for x in (k, v)]
    for kk, vv in ((grad[0], v), (k, grad[1])):
        for call in (lambda: at.decode_attention(q, kk, vv, table, n), lambda: at.window_attention(q, kk, vv, table, n, cu),
                     lambda: kc.write_kv(new, new, kk, vv, table, n),
                     lambda: kc.fork_pages(kk[None], vv[None], table, n, count, n - n),
                     lambda: kc.compact_pages(kk[None], vv[None], table, n, count)):
            with pytest.raises(RuntimeError, match="no backward"):
                call()
            with torch.no_grad():
                call()


def test_forward_mode_tangents_are_refused():
    rs = np.random.RandomState(2)
    k, v, table, n = make(rs, [40, 20], 2, 16, 64, torch.float16)
    q = torch.randn(2, 4, 64, device=DEV).half()
    cu = torch.arange(3, dtype=torch.int32, device=DEV)
    x, s = torch.randn(1, 2, 50, device=DEV), torch.zeros(1, 2, device=DEV)
    with fwd.dual_level():
        dual = [fwd.make_dual(t, torch.ones_like(t)) for t in (q, k, v, x, s)]
        for call in (lambda: at.decode_attention(dual[0], k, v, table, n), lambda: at.decode_attention(q, dual[1], v, table, n),
                     lambda: at.window_attention(dual[0], k, v, table, n, cu),
                     lambda: at.window_attention(q, k, dual[2], table, n, cu),
                     lambda: kc.write_kv(dual[0][:, :2], q[:, :2], k, v, table, n),
                     lambda: beam_select(dual[3], s), lambda: beam_select(x, dual[4])):
            with pytest.raises(RuntimeError, match="no .*derivative"):
                call()
    beam_select(x, s)


@pytest.mark.parametrize("page,dim,heads,what", [(512, 64, 4, "page size"), (8, 64, 4, "page size"), (24, 64, 4, "page size"),
                                                 (16, 136, 4, "head dimension"), (16, 60, 4, "head dimension"),
                                                 (16, 64, 1 << 21, "too many")])
def test_refusals_name_what_is_wrong(page, dim, heads, what):
    k = torch.zeros(2, 2, page, dim, device=DEV, dtype=torch.float16)
    q = torch.zeros(1, 1, dim, device=DEV, dtype=torch.float16).expand(1, heads, dim)
    table, n = (torch.zeros(s, dtype=torch.int32, device=DEV) for s in ((1, 3), (1,)))
    for call in (lambda: at.decode_attention(q, k, k, table, n), lambda: at.window_attention(q, k, k, table, n, offsets([1]))):
        with pytest.raises(NotImplementedError, match=what):
            call()


@pytest.mark.parametrize("axis", [0, 1])
def test_queries_broadcast_along_an_axis(axis):
    """A query that all tokens, or all heads, share is read where it is."""
    rs = np.random.RandomState(5)
    k, v, table, n = make(rs, [77, 300], 2, 32, 64, torch.float16)
    q = torch.randn((1, 8, 64) if axis == 0 else (60, 1, 64), device=DEV).half().expand(60, 8, 64)
    got = at.window_attention(q, k, v, table, n, offsets([20, 40]), return_lse=True)
    check(got, exact(q, k, v, table, n, [20, 40], 0, 0), torch.float16, True)
    got = at.decode_attention(q[:2], k, v, table, n, return_lse=True)
    check(got, exact(q[:2], k, v, table, n, [1, 1], 0, 0), torch.float16, False)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,past,q_heads,kv_heads,page,dim", [
    (8, 15000, 8, 1, 64, 128), (3, 9000, 6, 2, 16, 96), (70, 2500, 8, 2, 32, 64), (1100, 3000, 4, 1, 128, 128)])
def test_long_rows_to_their_own_rounding(new, past, q_heads, kv_heads, page, dim, dtype):
    """Over n keys an output is about n^(-1/2), so the tolerance has to be this case's own.
    With u as elsewhere, p the softmax and v the values: the output's rounding is u |o|; the
    n roundings of weights are independent, at most u p each and even within that, so their
    sum has a deviation below u (sum p^2 v^2 / 3)^(1/2), taken six times; a float16 weight
    below its normal range is off by 2^-25 at most where the largest is 2^6 or more, so all
    together by n 2^-31 max |v|; and float32 sums as elsewhere, 1e-4 sum p |v|.  That the
    tolerance is narrow enough shows in outputs without the values of 256 keys."""
    rs = np.random.RandomState(new)
    n = new + past
    k, v, table, lengths = make(rs, [n], kv_heads, page, dim, dtype)
    q = torch.randn(new, q_heads, dim, device=DEV).to(dtype)
    kk, vv = (x[table[0].long()].transpose(1, 2).reshape(-1, kv_heads, dim)[:n].double().repeat_interleave(q_heads // kv_heads, 1)
              for x in (k, v))
    s = torch.einsum("thd,nhd->htn", q.double(), kk) * dim ** -0.5
    p = s.masked_fill(torch.arange(n, device=DEV) > past + torch.arange(new, device=DEV)[:, None], -torch.inf).softmax(-1)
    o = torch.einsum("htn,nhd->thd", p, vv)
    deviation = (torch.einsum("htn,nhd->thd", p * p, vv * vv) / 3).sqrt()
    u = 2.0 ** -11 if dtype is torch.float16 else 2.0 ** -8
    tol = u * o.abs() + 6 * u * deviation + 1e-4 * torch.einsum("htn,nhd->thd", p, vv.abs())
    if dtype is torch.float16:
        tol += n * 2.0 ** -31 * vv.abs().max()
    for at_key in (0, n // 2 // 256 * 256, past - 256):
        part = slice(at_key, at_key + 256)
        assert bool((torch.einsum("htn,nhd->thd", p[..., part], vv[part]).abs() > tol).any(-1).float().mean() > 0.9)
    err = (at.window_attention(q, k, v, table, lengths, offsets([new])).double() - o).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("window", [1, 4, 31, 32, 64, 70])
def test_values_not_seen_at_every_place_of_a_window(window):
    """The token whose window begins at the row's second key, and its neighbours, too."""
    rs = np.random.RandomState(window)
    n, dim = 150, 64
    k, v, table, lengths = make(rs, [n], 1, 16, dim, torch.float16)
    q = torch.randn(n, 4, dim, device=DEV).half()
    want = exact(q, k, v, table, lengths, [n], window, 0)
    pos = torch.arange(n, device=DEV)
    for place in (0, 1, window - 1, window, window + 1, 2 * window, n - 1):
        w = v.clone()
        w[int(table[0, place // 16]), :, place % 16, 5] = float("nan")
        out = at.window_attention(q, k, w, table, lengths, offsets([n]), window=window, return_lse=True)
        hit = torch.zeros(n, 4, dim, dtype=torch.bool, device=DEV)
        hit[:, :, 5] = ((place <= pos) & (place > pos - window))[:, None]
        assert out[0][hit].isnan().all()
        check((out[0].masked_fill(hit, 0), out[1]), (want[0].masked_fill(hit, 0), *want[1:]), torch.float16, weights=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new,heads", [(1, 2), (40, 2), (300, 80)])  # the last has whole rows, not shares of the keys
def test_scores_that_grow_along_the_row_and_large_values(new, heads, dtype):
    """Scores that rise by 80 over the row: the weights' reference lags behind them, and must
    not lag so far that a weight times a large value passes float32's range."""
    rs = np.random.RandomState(new)
    n, dim = 1500, 64
    k, v, table, lengths = make(rs, [n], heads, 16, dim, dtype)
    v *= 1e20 if dtype is torch.bfloat16 else 1e3
    for place in range(n):
        k[int(table[0, place // 16]), :, place % 16, 0] = 40.0 * place / n  # times 16 / 8: up to 80
    q = torch.randn(new, heads, dim, device=DEV).to(dtype)
    q[:, :, 0] = 16.0
    want = exact(q, k, v, table, lengths, [new], 0, 0)
    check(at.window_attention(q, k, v, table, lengths, offsets([new]), return_lse=True), want, dtype, True)
    one = [x[-1:] for x in want]
    check(at.decode_attention(q[-1:], k, v, table, lengths, return_lse=True), one, dtype, False)


def test_rows_summed_again_do_not_run_into_the_wait_limit():
    """Many such rows keep their warps far beyond a wait's limit: as long as they come along,
    the others wait on.  A model whose values are NaN throughout is not summed again at all."""
    rs = np.random.RandomState(3)
    new, n, heads, dim = 512, 4096, 64, 128
    k, v, table, lengths = make(rs, [n], heads, 64, dim, torch.float16)
    q = torch.randn(new, 8 * heads, dim, device=DEV).half()
    lib = N.lib()

    def run(values):
        return at.window_attention(q, k, values, table, lengths, offsets([new]))

    clean, w = run(v), v.clone()
    place = n - 130  # the tokens before it, in its tile, do not see it
    w[int(table[0, place // 64]), :, place % 64, 9] = float("inf")
    kc.check_device()
    try:
        assert lib.qs_set_wait_limit_ns(3_000_000) == N.QS_OK
        got = run(w)
        kc.check_device()
        gone = run(torch.full_like(v, float("nan")))
        kc.check_device()
    finally:
        lib.qs_set_wait_limit_ns(0)
    hit = torch.arange(n - new, n, device=DEV) >= place
    assert gone.isnan().all() and not got[hit, :, 9].isfinite().any()
    keep = torch.arange(dim, device=DEV) != 9
    assert torch.equal(got[..., keep], clean[..., keep])
    # weights rounded in one sum and not in the other: 2^-11 of the sum of p |v|, below 1, and the outputs' own rounding
    assert float((got[~hit, :, 9].float() - clean[~hit, :, 9].float()).abs().max()) < 2.0 ** -9
