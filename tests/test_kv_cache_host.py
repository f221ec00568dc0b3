"""Refusals of the decoding operators (no GPU): what is checked before anything is launched."""
import ctypes

import pytest
import torch

from quipsharp_b200 import _native as N
from quipsharp_b200 import attention, beam, kv_cache as kc


def pool(**change):
    p = N.KVPool()
    base = dict(k=4096, v=8192, dtype=N.QS_F16, layers=1, pages=4, heads=2, page=16, dim=64)
    for name, value in {**base, **change}.items():
        if not name.endswith("stride"):
            setattr(p, name, value)
    p.k_stride[:] = change.get("k_stride", (0, 2048, 1024, 64))
    p.v_stride[:] = change.get("v_stride", (0, 2048, 1024, 64))
    return p


def test_struct_matches_the_header():
    assert ctypes.sizeof(N.KVPool) == 16 + 8 + 5 * 8 + 8 * 8


@pytest.mark.parametrize("change,status", [
    (dict(dtype=N.QS_F32), N.QS_ERR_INVALID_ARG), (dict(pages=0), N.QS_ERR_INVALID_ARG), (dict(k=None), N.QS_ERR_INVALID_ARG),
    (dict(page=24), N.QS_ERR_UNSUPPORTED), (dict(page=8), N.QS_ERR_UNSUPPORTED), (dict(page=512), N.QS_ERR_UNSUPPORTED),
    (dict(dim=36), N.QS_ERR_UNSUPPORTED), (dict(dim=264), N.QS_ERR_UNSUPPORTED), (dict(v=8200), N.QS_ERR_ALIGNMENT),
    (dict(k_stride=(0, 2048, 1024, 60)), N.QS_ERR_ALIGNMENT), (dict(pages=(1 << 28) + 1), N.QS_ERR_UNSUPPORTED)])
def test_pools_are_checked(change, status):
    lib, p = N.lib(), pool(**change)
    one = ctypes.c_void_p(256)
    assert lib.qs_cache_write(N.ref(p), 0, 1, None, None, None, None, 64, 64, None, 64, 64, 0, None) == status
    assert lib.qs_cache_fork(N.ref(p), 1, 1, one, one, one, one, one, one, one, one, 1 << 20, None) == status
    assert lib.qs_attn_decode(None, 64, 64, N.ref(p), 0, 2, 1, None, None, 1.0, 0, 0, None, None, None, 0, None) == status


def test_cache_arguments():
    lib, p, at = N.lib(), pool(), ctypes.c_void_p
    need = lib.qs_cache_workspace_bytes(1, 4)
    assert need > 0 and lib.qs_cache_workspace_bytes(8193, 4) == -1 and lib.qs_cache_workspace_bytes(1, 0) == -1

    def fork(table_out=at(2560), ws=at(1 << 16), nb=need, rows=1, parents=at(1024)):
        return lib.qs_cache_fork(N.ref(p), rows, 1, at(256), at(512), at(768), parents, table_out, at(2816), at(3584), ws, nb,
                                 None)

    assert fork(parents=None) == N.QS_ERR_INVALID_ARG
    assert fork(table_out=at(256)) == N.QS_ERR_INVALID_ARG and b"overlap" in lib.qs_last_error()
    assert fork(nb=need - 1) == N.QS_ERR_WORKSPACE and fork(ws=None) == N.QS_ERR_WORKSPACE
    assert fork(ws=at((1 << 16) + 8)) == N.QS_ERR_ALIGNMENT
    assert fork(rows=9000) == N.QS_ERR_UNSUPPORTED and fork(rows=-1) == N.QS_ERR_INVALID_ARG
    assert lib.qs_cache_extend(20, 4, 1, 1, at(256), at(512), at(768), at(1024), at(256), at(512), at(768), at(1 << 16), need,
                               None) == N.QS_ERR_UNSUPPORTED
    assert lib.qs_cache_write(N.ref(p), 2, 1, at(256), at(512), None, at(4096), 128, 64, at(4096), 128, 64, 3,
                              None) == N.QS_ERR_INVALID_ARG  # one token per row without cu
    assert lib.qs_cache_write(N.ref(p), 2, 1, at(256), at(512), at(768), at(4100), 128, 64, at(4096), 128, 64, 3,
                              None) == N.QS_ERR_ALIGNMENT
    assert lib.qs_cache_write(N.ref(p), 2, 1, at(256), at(512), at(768), None, 128, 64, None, 128, 64, 0, None) == N.QS_OK


def test_attention_arguments():
    lib, p, at = N.lib(), pool(), ctypes.c_void_p
    sizes = lib.qs_attn_decode_workspace_bytes
    need = sizes(3, 4, 2, 64, 16, 400, 0, 0)
    assert need > 0 and sizes(3, 4, 2, 64, 16, 10, 0, 0) == sizes(3, 4, 2, 64, 16, 100, 500, 4) == 0  # few keys: no joins
    assert sizes(3, 5, 2, 64, 16, 100, 0, 0) == sizes(3, 4, 2, 136, 16, 100, 0, 0) == sizes(3, 4, 2, 64, 16, -1, 0, 0) == -1

    def decode(q=at(4096), heads=4, scale=0.1, window=0, sinks=0, ws=at(1 << 16), nb=need, pool=p, q_head=64):
        return lib.qs_attn_decode(q, 256, q_head, N.ref(pool), 3, heads, 400, at(256), at(512), scale, window, sinks, at(8192),
                                  None, ws, nb, None)

    assert decode(q=None) == N.QS_ERR_INVALID_ARG and decode(heads=5) == N.QS_ERR_INVALID_ARG
    assert decode(scale=0.0) == decode(scale=float("nan")) == decode(scale=float("inf")) == N.QS_ERR_INVALID_ARG
    assert decode(window=-1) == decode(sinks=-1) == N.QS_ERR_INVALID_ARG
    assert decode(nb=need - 1) == N.QS_ERR_WORKSPACE and decode(ws=at(264)) == N.QS_ERR_ALIGNMENT
    assert decode(q=at(4098)) == decode(q_head=66) == N.QS_ERR_ALIGNMENT
    assert decode(pool=pool(dim=136)) == N.QS_ERR_UNSUPPORTED
    assert lib.qs_attn_window(at(4096), 256, 64, N.ref(p), 3, 1, 4, 1, at(256), at(512), None, 0.1, 0, 0, at(8192), None, None,
                              0, None) == N.QS_ERR_INVALID_ARG
    assert lib.qs_attn_window(at(4096), 256, 64, N.ref(p), 3, 1, 2 * 129, 1, at(256), at(512), at(768), 0.1, 0, 0, at(8192),
                              None, None, 0, None) == N.QS_ERR_UNSUPPORTED


def test_beam_arguments():
    lib, at = N.lib(), ctypes.c_void_p
    need = lib.qs_beam_workspace_bytes(2, 4, 1000, 4)
    assert need > 0
    for args in ((2, 65, 1000, 4), (2, 4, 1000, 65), (2, 4, 3, 4), (2, 0, 10, 1), (2, 4, 1000, 0)):
        assert lib.qs_beam_workspace_bytes(*args) == -1

    def select(dtype=N.QS_F32, beams=4, vocab=1000, n=4, logits=at(4096), ws=at(1 << 16), nb=need, scores=at(256)):
        return lib.qs_beam_select(logits, dtype, 4000, 1000, 2, beams, vocab, scores, None, n, 0, at(512), at(768), at(1024),
                                  ws, nb, None)

    assert select(dtype=N.QS_I32) == select(n=0) == select(n=1001) == select(scores=None) == N.QS_ERR_INVALID_ARG
    assert select(beams=65) == select(n=65) == N.QS_ERR_UNSUPPORTED
    assert select(logits=at(4098)) == select(ws=at(264)) == N.QS_ERR_ALIGNMENT
    assert select(nb=need - 1) == N.QS_ERR_WORKSPACE


def test_python_refusals():
    table, n, c = (torch.zeros(s, dtype=torch.int32) for s in ((2, 3), (2,), (4,)))
    k = torch.zeros(1, 4, 2, 16, 64, dtype=torch.float16)
    q = torch.zeros(2, 4, 64, dtype=torch.float16)
    for call in (lambda: kc.fork_pages(k, k, table, n, c, n), lambda: kc.compact_pages(k, k, table, n, c),
                 lambda: kc.extend_pages(table, n, c, n, 16), lambda: kc.write_kv(q[:, :2], q[:, :2], k[0], k[0], table, n),
                 lambda: attention.decode_attention(q, k[0], k[0], table, n),
                 lambda: beam.beam_select(torch.zeros(1, 2, 9), torch.zeros(1, 2))):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
    with pytest.raises(RuntimeError, match="no backward"):
        attention._arguments("decode_attention", q.float().requires_grad_(), k[0], k[0], table, n, None, 0, None)
    with pytest.raises(RuntimeError, match="no backward"):
        beam.beam_select(torch.zeros(1, 2, 9, requires_grad=True), torch.zeros(1, 2))
    for bad, error in ((dict(q=q.float()), TypeError), (dict(q=q[..., :32]), ValueError), (dict(q=q[:, :3]), ValueError),
                       (dict(window=0), ValueError), (dict(sinks=-1), ValueError), (dict(lengths=n.long()), TypeError),
                       (dict(lengths=n[:1]), ValueError), (dict(k=k), ValueError), (dict(v=k[0].bfloat16()), TypeError)):
        a = dict(q=q, k=k[0], v=k[0], table=table, lengths=n, window=None, sinks=0, scale=None)
        a.update(bad)
        with pytest.raises(error):
            attention._arguments("decode_attention", a["q"], a["k"], a["v"], a["table"], a["lengths"], a["window"], a["sinks"],
                                 a["scale"])
    with pytest.raises(TypeError):
        kc.PagedKVCache(1, 1, 64, 4, 1, 64, dtype=torch.float32)
    with pytest.raises(NotImplementedError):
        kc.PagedKVCache(1, 1, 64, 4, 1, 64, page_size=24)
    with pytest.raises(NotImplementedError):
        kc.PagedKVCache(1, 1, 65, 4, 1, 64)
    with pytest.raises(ValueError):
        kc.PagedKVCache(1, 1, 64, 0, 1, 64)


def test_views_are_read_in_place_where_they_can_be():
    x = torch.zeros(4, 6, 64, dtype=torch.float16)
    assert N.rows_of_8(x[:, 2:4]) .data_ptr() == x[:, 2:4].data_ptr()
    odd = torch.zeros(4, 65, dtype=torch.float16)[:, :64]
    assert N.rows_of_8(odd).stride() == (64, 1)
    assert N.rows_of_8(x.transpose(1, 2)).is_contiguous()
