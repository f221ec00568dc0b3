"""More refusals of the decoding operators (no GPU; see test_kv_cache_host)."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from quipsharp_b200 import attention, beam


def test_pools_without_a_key_head():
    q, k = torch.zeros(2, 4, 64, dtype=torch.float16), torch.zeros(4, 0, 16, 64, dtype=torch.float16)
    table, n = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="0 key heads"):
        attention._arguments("decode_attention", q, k, k, table, n, None, 0, None)


def test_forward_mode_tangents():
    with fwd.dual_level():
        x = fwd.make_dual(torch.zeros(1, 2, 9), torch.ones(1, 2, 9))
        with pytest.raises(RuntimeError, match="no forward-mode"):
            beam.beam_select(x, torch.zeros(1, 2))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        beam.beam_select(x, torch.zeros(1, 2))


@pytest.mark.parametrize("pad", [1 << 31, -(1 << 31) - 1, 1 << 40])
def test_padding_tokens_are_int32(pad):
    with pytest.raises(ValueError, match="int32"):
        beam.beam_select(torch.zeros(1, 2, 9), torch.zeros(1, 2), pad=pad)


def test_windows_of_any_size():
    """A number past 64 bits is a very large one, not what is left of it."""
    q, k = torch.zeros(2, 4, 64, dtype=torch.float16), torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    table, n = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    *_, window, sinks = attention._arguments("decode_attention", q, k, k, table, n, (1 << 64) + 5, (1 << 65) + 1, None)
    assert 1 << 31 < window < 1 << 63 and 1 << 31 < sinks < 1 << 63
