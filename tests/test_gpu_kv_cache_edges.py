"""Page moves of the key-value cache at the edges of what tables and arguments may hold."""
import threading

import numpy as np
import pytest
import torch

from quipsharp_b200 import _native as N
from quipsharp_b200 import kv_cache as kc
from test_gpu_kv_cache import DEV, on, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [1, 3, 40])
def test_write_leaves_out_tokens_before_the_first_row(first):
    """cu[0] > 0, as of a slice of a larger batch: the tokens before it belong to no row, and
    what the cache held stays."""
    page = 16
    g = torch.Generator(device=DEV).manual_seed(first)
    k, v = (torch.randn(6, 2, page, 8, generator=g, device=DEV).half() for _ in range(2))
    kn, vn = (torch.randn(first + 9, 2, 8, generator=g, device=DEV).half() for _ in range(2))
    table, lengths, cu = on(np.array([[4, 1], [2, 5]], np.int32), np.array([22, 7], np.int32),
                            np.array([first, first + 5, first + 9], np.int32))
    wk, wv = k.clone(), v.clone()
    for w, new in ((wk, kn), (wv, vn)):
        for row, n, at, count in ((0, 22, first, 5), (1, 7, first + 5, 4)):
            for j in range(count):
                pos = n - count + j
                w[int(table[row, pos // page]), :, pos % page] = new[at + j]
    kc.write_kv(kn, vn, k, v, table, lengths, cu)
    same(k, wk.cpu(), "keys"), same(v, wv.cpu(), "values")


@pytest.mark.parametrize("rows,pages", [(4, 6), (4, 40000), (8000, 8000)])
def test_children_of_a_row_whose_last_page_is_absent(rows, pages):
    """A part-filled page that was never found (-1) is absent in every child: no page is taken
    for it, and nothing becomes visible in its place."""
    page = 16
    k, v = (torch.randn(1, pages, 1, page, 8, device=DEV).half() for _ in range(2))
    table = np.full((rows, 3), -1, np.int32)
    table[0, 0], table[1, :2] = 2, (3, 0)
    lengths = np.zeros(rows, np.int32)
    lengths[:2] = 20, 25
    refcount = np.zeros(pages, np.int32)
    refcount[[2, 3, 0]] = 1
    parents = np.full(rows, -1, np.int32)
    parents[:4] = 0, 0, 1, 1
    wk, wv = k.clone(), v.clone()
    for w in (wk, wv):
        w[:, 1, :, :9] = w[:, 0, :, :9]
    t, n, c = kc.fork_pages(k, v, *on(table, lengths, refcount, parents))
    assert t[:4].tolist() == [[2, -1, -1], [2, -1, -1], [3, 0, -1], [3, 1, -1]] and bool((t[4:] == -1).all())
    assert n[:4].tolist() == [20, 20, 25, 25] and c[:6].tolist() == [1, 1, 2, 2, 0, 0] and int(c.sum()) == 6
    same(k, wk.cpu(), "keys"), same(v, wv.cpu(), "values")
    kc.check_device()


def test_caches_of_different_sizes_in_two_threads():
    """Each call lets its kernel have shared memory and launches: another thread's smaller call
    in between must not take that away."""
    lib = N.lib()
    calls = []
    for pages in (19000, 7000):
        state = on(np.full((4, 4), -1, np.int32), np.zeros(4, np.int32), np.zeros(pages, np.int32), np.ones(4, np.int32))
        out = [t.clone() for t in state[:3]]
        nb = lib.qs_cache_workspace_bytes(4, pages)
        ws = torch.empty(nb, dtype=torch.uint8, device=DEV)
        calls.append((state, out, ws, (16, pages, 4, 4, *(t.data_ptr() for t in (*state, *out, ws)), nb,
                                       torch.cuda.Stream().cuda_stream)))
    torch.cuda.synchronize()
    failed = [0, 0]

    def work(i):
        for _ in range(4000):
            if lib.qs_cache_extend(*calls[i][3]) != N.QS_OK:
                failed[i] += 1

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert failed == [0, 0]
    for _, (table, lengths, count), _, _ in calls:
        assert table[:, 0].tolist() == [0, 1, 2, 3] and lengths.tolist() == [1] * 4 and int(count.sum()) == 4
    kc.check_device()


def test_errors_of_two_kinds_are_both_reported():
    """One call finds a token count out of range and no free page: two checks raise, a third does not."""
    args = on(np.array([[0], [-1]], np.int32), np.array([16, 0], np.int32), np.array([1], np.int32), np.array([-1, 5], np.int32))
    kc.check_device()
    kc.extend_pages(*args, 16)
    with pytest.raises(RuntimeError, match="no free page"):
        kc.check_device()
    with pytest.raises(IndexError):
        kc.check_device()
    kc.check_device()
