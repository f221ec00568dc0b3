"""Page moves of the key-value cache against a plain host implementation: page
numbers, counts and copied contents have to be equal, bit for bit."""
import numpy as np
import pytest
import torch

from quipsharp_b200 import kv_cache as kc

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make_state(rs, rows, page, pages, width, max_len, share=1):
    """Tables of `rows` rows in groups of `share` that hold the same whole pages."""
    table = np.full((rows, width), -1, np.int32)
    lengths = np.zeros(rows, np.int32)
    free = list(rs.permutation(pages))
    for g in range(0, rows, share):
        n = int(rs.randint(0, max_len + 1))
        whole = (n // page) if share > 1 else 0
        common = [free.pop() for _ in range(whole)]
        for i in range(g, min(rows, g + share)):
            lengths[i] = n
            used = -(-n // page)
            table[i, :used] = common + [free.pop() for _ in range(used - whole)]
    refcount = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    return table, lengths, refcount


def pools(rs, layers, pages, heads, page, dim, dtype):
    g = torch.Generator().manual_seed(int(rs.randint(1 << 30)))
    return [torch.randn(layers, pages, heads, page, dim, generator=g).to(dtype) for _ in range(2)]


def fork_host(k, v, table, lengths, refcount, parents, page):
    k, v = k.clone(), v.clone()
    rows, width = table.shape
    new, n, count = np.full_like(table, -1), np.zeros_like(lengths), refcount.astype(np.int64).copy()
    for i in range(rows):  # references that go
        for p in table[i, :-(-int(lengths[i]) // page)]:
            if p >= 0:
                count[p] -= 1
    first, copies = {}, []
    for i in range(rows):
        p = int(parents[i])
        if p < 0 or p >= rows:
            continue
        n[i] = lengths[p]
        used = -(-int(n[i]) // page)
        new[i, :used] = table[p, :used]
        if p in first and n[i] % page:
            copies.append(i)
            new[i, used - 1] = -1
        first.setdefault(p, i)
        for q in new[i, :used]:
            if q >= 0:
                count[q] += 1
    free = [q for q in range(len(count)) if count[q] == 0]
    for r, i in enumerate(copies):
        last, fill = int(n[i]) // page, int(n[i]) % page
        if r >= len(free):
            continue
        src, dst = int(table[parents[i], last]), free[r]
        new[i, last], count[dst] = dst, 1
        k[:, dst, :, :fill], v[:, dst, :, :fill] = k[:, src, :, :fill], v[:, src, :, :fill]
    return k, v, new, n, count.astype(np.int32)


def on(*arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)).to(DEV) for a in arrays]


def same(got, want, what):
    assert torch.equal(got.cpu(), torch.as_tensor(want)), what


@pytest.mark.parametrize("rows,share,page,pages,max_len,heads,dim,layers,dtype", [
    (4, 4, 16, 96, 200, 4, 64, 2, torch.float16),
    (1, 1, 16, 8, 40, 1, 8, 1, torch.bfloat16),
    (24, 8, 32, 300, 500, 3, 80, 3, torch.bfloat16),
    (600, 5, 16, 6000, 150, 1, 16, 1, torch.float16),      # more rows than threads of a block
    (40, 4, 16, 40000, 900, 1, 8, 1, torch.float16),       # more pages than one block scans: the cluster
    (8192, 2, 16, 16000, 15, 1, 8, 1, torch.bfloat16),     # one block whose counts do not fit shared memory
])
@pytest.mark.parametrize("kind", ["random", "identity", "all_of_one", "free_all"])
def test_fork(rows, share, page, pages, max_len, heads, dim, layers, dtype, kind):
    rs = np.random.RandomState(rows + page)
    width = -(-max_len // page) + 1
    table, lengths, refcount = make_state(rs, rows, page, pages, width, max_len, share)
    parents = {"random": rs.randint(-1, rows, rows), "identity": np.arange(rows), "all_of_one": np.full(rows, rows // 2),
               "free_all": np.full(rows, -1)}[kind].astype(np.int32)
    k, v = pools(rs, layers, pages, heads, page, dim, dtype)
    wk, wv, wt, wn, wc = fork_host(k, v, table, lengths, refcount, parents, page)
    k, v = k.to(DEV), v.to(DEV)
    t, n, c = kc.fork_pages(k, v, *on(table, lengths, refcount, parents))
    same(t, wt, "table"), same(n, wn, "lengths"), same(c, wc, "refcount"), same(k, wk, "keys"), same(v, wv, "values")
    kc.check_device()


def test_fork_keeps_the_callers_references():
    """A count above the table's references (a prefix that the caller holds) is never freed."""
    page, pages = 16, 8
    k, v = (torch.randn(1, pages, 1, page, 8, device=DEV).half() for _ in range(2))
    table, lengths, refcount = on(np.array([[3, 5]], np.int32), np.array([20], np.int32),
                                  np.array([0, 0, 0, 2, 0, 1, 0, 0], np.int32))
    t, n, c = kc.fork_pages(k, v, table, lengths, refcount, on(np.array([-1], np.int32))[0])
    assert c.tolist() == [0, 0, 0, 1, 0, 0, 0, 0] and n.tolist() == [0] and t.tolist() == [[-1, -1]]


def test_fork_of_pools_in_token_major_order():
    """Pools whose head and token axes are exchanged (a transposed view) copy the same rows."""
    rs = np.random.RandomState(5)
    page, pages, rows = 16, 60, 6
    table, lengths, refcount = make_state(rs, rows, page, pages, 8, 100, 3)
    parents = np.array([1, 1, 1, 4, -1, 4], np.int32)
    k, v = pools(rs, 2, pages, 3, page, 24, torch.bfloat16)
    wk, wv, wt, _, _ = fork_host(k, v, table, lengths, refcount, parents, page)
    kt, vt = (x.to(DEV).transpose(2, 3).contiguous().transpose(2, 3) for x in (k, v))
    t, _, _ = kc.fork_pages(kt, vt, *on(table, lengths, refcount, parents))
    same(t, wt, "table"), same(kt, wk, "keys"), same(vt, wv, "values")


def test_fork_without_free_pages_reports_and_recovers():
    page, pages = 16, 2
    k, v = (torch.randn(1, pages, 1, page, 8, device=DEV).half() for _ in range(2))
    args = on(np.array([[0, 1], [-1, -1], [-1, -1]], np.int32), np.array([20, 0, 0], np.int32), np.array([1, 1], np.int32))
    t, n, c = kc.fork_pages(k, v, *args, on(np.array([0, 0, -1], np.int32))[0])
    assert t.tolist() == [[0, 1], [0, -1], [-1, -1]] and c.tolist() == [2, 1] and n.tolist() == [20, 20, 0]
    with pytest.raises(RuntimeError, match="no free page"):
        kc.check_device()
    kc.check_device()  # the read cleared it
    kc.fork_pages(k, v, *args, on(np.array([7, 0, -2], np.int32))[0])
    with pytest.raises(IndexError):
        kc.check_device()


@pytest.mark.parametrize("rows,page,pages,max_len,heads,dim,layers", [
    (5, 16, 200, 300, 2, 64, 2), (1, 64, 3, 10, 1, 128, 1), (30, 32, 40000, 700, 1, 8, 1), (9, 16, 64, 90, 3, 40, 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(rows, page, pages, max_len, heads, dim, layers, in_place):
    rs = np.random.RandomState(pages)
    table, lengths, refcount = make_state(rs, rows, page, pages, -(-max_len // page) + 2, max_len)
    k, v = pools(rs, layers, pages, heads, page, dim, torch.float16)
    used = np.flatnonzero(refcount)
    src, dst = used[used >= len(used)], np.setdiff1d(np.arange(len(used)), used)
    to = np.arange(pages)
    to[src] = dst
    wt = np.where(table >= 0, to[np.maximum(table, 0)], -1)
    wc = (np.arange(pages) < len(used)).astype(np.int32)
    wk, wv = k.clone(), v.clone()
    wk[:, dst], wv[:, dst] = k[:, src], v[:, src]
    k, v = k.to(DEV), v.to(DEV)
    if in_place:
        cache = kc.PagedKVCache(layers, heads, dim, pages, rows, (-(-max_len // page) + 2) * page, page, torch.float16)
        cache.k, cache.v, (cache.table, cache.lengths, cache.refcount) = k, v, on(table, lengths, refcount)
        n = cache.compact()
        t, c = cache.table, cache.refcount
    else:
        t, c, n = kc.compact_pages(k, v, *on(table, lengths, refcount))
    assert n.tolist() == [len(used)]
    same(t, wt.astype(np.int32), "table"), same(c, wc, "refcount"), same(k, wk, "keys"), same(v, wv, "values")


def test_compact_of_an_empty_and_of_a_full_pool():
    for table, lengths, refcount in (([[-1]], [0], [0, 0]), ([[1, 0]], [32], [1, 1])):
        k, v = (torch.randn(1, 2, 1, 16, 8, device=DEV).half() for _ in range(2))
        args = on(np.array(table, np.int32), np.array(lengths, np.int32), np.array(refcount, np.int32))
        t, c, n = kc.compact_pages(k, v, *args)
        assert t.tolist() == table and c.tolist() == refcount and n.tolist() == [sum(refcount)]


@pytest.mark.parametrize("rows,page,pages,max_len,max_new,heads,dim", [
    (16, 16, 1400, 700, 512, 8, 128), (1, 256, 2, 0, 300, 1, 8), (700, 16, 40000, 60, 1, 2, 72), (3, 64, 50, 200, 0, 1, 64),
    (9, 16, 25000, 300, 70, 1, 16)])
def test_extend_and_write(rows, page, pages, max_len, max_new, heads, dim):
    rs = np.random.RandomState(rows)
    width = -(-(max_len + max_new) // page) + 1
    table, lengths, refcount = make_state(rs, rows, page, pages, width, max_len)
    new = rs.randint(0, max_new + 1, rows).astype(np.int32)
    wt, wc = table.copy(), refcount.copy()
    free = iter(np.flatnonzero(refcount == 0))
    for i in range(rows):
        for c in range(-(-int(lengths[i]) // page), -(-int(lengths[i] + new[i]) // page)):
            wt[i, c] = next(free)
            wc[wt[i, c]] = 1
    t, n, c = kc.extend_pages(*on(table, lengths, refcount, new), page)
    same(t, wt, "table"), same(n, lengths + new, "lengths"), same(c, wc, "refcount")
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    k, v = pools(rs, 1, pages, heads, page, dim, torch.bfloat16)
    fused = torch.randn(int(cu[-1]), 3 * heads, dim).bfloat16()  # keys and values as views of a joint projection
    kn, vn = fused[:, heads:2 * heads], fused[:, 2 * heads:]
    wk, wv = k.clone(), v.clone()
    for i in range(rows):
        for j in range(new[i]):
            pos = lengths[i] + j
            wk[0, wt[i, pos // page], :, pos % page] = kn[cu[i] + j]
            wv[0, wt[i, pos // page], :, pos % page] = vn[cu[i] + j]
    k, v, fused = k.to(DEV), v.to(DEV), fused.to(DEV)
    kc.write_kv(fused[:, heads:2 * heads], fused[:, 2 * heads:], k[0], v[0], t, n, on(cu)[0])
    same(k, wk, "keys"), same(v, wv, "values")
    kc.check_device()


def test_extend_past_the_pool_and_the_line():
    page = 16
    t, n, c = kc.extend_pages(*on(np.array([[1, -1], [-1, -1]], np.int32), np.array([10, 0], np.int32),
                                  np.array([0, 1], np.int32), np.array([30, 5], np.int32)), page)
    # row 0 wants two more pages and has room for one: page 0; row 1 finds none
    assert t.tolist() == [[1, 0], [-1, -1]] and n.tolist() == [40, 5] and c.tolist() == [1, 1]
    with pytest.raises(RuntimeError, match="no free page"):
        kc.check_device()
    k, v = (torch.zeros(2, 1, page, 8, device=DEV, dtype=torch.float16) for _ in range(2))
    new = torch.ones(35, 1, 8, device=DEV, dtype=torch.float16)
    kc.write_kv(new, new, k, v, t, n, on(np.array([0, 30, 35], np.int32))[0])  # tokens without a page are left out
    assert k.sum().item() == v.sum().item() == (32 - 10) * 8
    kc.check_device()


def test_cache_object_steps_in_a_graph():
    """extend, write and fork keep their tensors in place, so a captured step can be replayed."""
    cache = kc.PagedKVCache(1, 2, 16, num_pages=64, rows=4, max_len=100, page_size=16, dtype=torch.float16)
    parents = torch.tensor([0, 0, 2, 2], dtype=torch.int32, device=DEV)
    new = torch.randn(4, 2, 16, device=DEV).half()

    def step():
        cache.fork(parents)
        cache.extend(1)
        cache.write(0, new, new)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(18):
        graph.replay()
    cache.check()
    assert cache.lengths.tolist() == [19] * 4  # capturing runs nothing
    assert cache.table[0, 0] == cache.table[1, 0] and cache.table[0, 1] != cache.table[1, 1]
    assert int(cache.refcount.sum()) == 8 and int((cache.refcount > 0).sum()) == 6
    got = cache.k[0, cache.table[3, 1].long(), :, 2]
    assert torch.equal(got, new[3])
    cache.free([0, 1, 2, 3])
    assert int(cache.refcount.sum()) == 0 and cache.lengths.tolist() == [0] * 4


def test_arguments_that_need_a_copy_or_a_refusal():
    rs = np.random.RandomState(3)
    page, pages = 16, 40
    state = make_state(rs, 4, page, pages, 6, 80)
    table, lengths, refcount = on(*state)
    parents = torch.tensor([1, 1, 3, -1], dtype=torch.int32, device=DEV)
    k, v = (x.to(DEV) for x in pools(rs, 2, pages, 2, page, 24, torch.float16))
    want = kc.fork_pages(k, v, table, lengths, refcount, parents)
    spread = torch.stack((parents, parents), -1)[:, 0]
    for a, b in zip(kc.fork_pages(k, v, table, lengths, refcount, spread), want):
        assert torch.equal(a, b)
    new = torch.tensor([3, 0, 20, 1], dtype=torch.int32, device=DEV)
    want = kc.extend_pages(table, lengths, refcount, new, page)
    for a, b in zip(kc.extend_pages(table, lengths, refcount, new, np.int64(page)), want):
        assert torch.equal(a, b)
    for error, call in (
            (TypeError, lambda: kc.fork_pages(k, v, table, lengths, refcount, parents.long())),
            (TypeError, lambda: kc.fork_pages(k.float(), v.float(), table, lengths, refcount, parents)),
            (ValueError, lambda: kc.fork_pages(k, v[:, :9], table, lengths, refcount, parents)),
            (ValueError, lambda: kc.fork_pages(k, v, table, lengths, refcount[:9], parents)),
            (ValueError, lambda: kc.compact_pages(k, v, table, lengths[:3], refcount)),
            (NotImplementedError, lambda: kc.extend_pages(table, lengths, refcount, new, 24)),
            (ValueError, lambda: kc.write_kv(k[0, 0], v[0, 0], k[0], v[0], table, lengths)),
            (RuntimeError, lambda: kc.fork_pages(k, v, table, lengths, refcount, parents.cpu()))):
        with pytest.raises(error):
            call()
