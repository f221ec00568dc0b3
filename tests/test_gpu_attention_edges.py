"""Attention over the paged cache at the edges of what a row, a table and a pool may hold
(see test_gpu_attention for the exact form and the tolerances)."""
import numpy as np
import pytest
import torch

from quipsharp_b200 import attention as at
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
