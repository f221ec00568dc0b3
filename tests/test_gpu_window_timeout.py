"""Bounded waits of the window attention kernel, without a GPU fault.  The warps that sum
wait for the first job; with tens of thousands of empty rows before the only one with
tokens, finding it takes longer than a barrier's own patience, so with the limit at 1 ns
that wait gives up: the kernel drains its own copies and products and returns, the status
comes back as QS_ERR_TIMEOUT once, and with the default limit the next call is right."""
import pytest
import torch

from quipsharp_b200 import _native as N
from quipsharp_b200 import attention as at
from quipsharp_b200 import kv_cache as kc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,past", [(700, 300), (5, 3000)])
def test_short_wait_limit_reports_timeout_then_recovers(new, past):
    page, dim, n, rows = 32, 128, new + past, 40000
    pages = -(-n // page)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(pages, 2, page, dim, generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn(new, 8, dim, generator=g, device="cuda").half()
    table = torch.full((rows, pages), -1, dtype=torch.int32, device="cuda")
    table[-1] = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).int().cuda()
    lengths, cu = (torch.zeros(rows + i, dtype=torch.int32, device="cuda") for i in range(2))
    lengths[-1], cu[-1] = n, new
    lib = N.lib()
    want = at.window_attention(q, k, v, table, lengths, cu)
    alone = at.window_attention(q, k, v, table[-1:], lengths[-1:], cu[-2:])
    # the number of rows decides whether the keys are split: equal up to the roundings of
    # weights and outputs, each 2^-11 of what it rounds
    assert float((want.float() - alone.float()).norm() / alone.float().norm()) < 4 * 2 ** -11
    kc.check_device("cuda")
    try:
        assert lib.qs_set_wait_limit_ns(1) == N.QS_OK
        at.window_attention(q, k, v, table, lengths, cu)
        assert lib.qs_device_status(N.stream_of(q)) == N.QS_ERR_TIMEOUT
        assert lib.qs_device_status(N.stream_of(q)) == N.QS_OK  # the read cleared it
    finally:
        lib.qs_set_wait_limit_ns(0)
    assert torch.equal(at.window_attention(q, k, v, table, lengths, cu), want)
    kc.check_device("cuda")
