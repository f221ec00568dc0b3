"""More refusals of the decoding operators (no GPU; see test_kv_cache_host)."""
import pytest
import torch

from quipsharp_b200 import attention


def test_pools_without_a_key_head():
    q, k = torch.zeros(2, 4, 64, dtype=torch.float16), torch.zeros(4, 0, 16, 64, dtype=torch.float16)
    table, n = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="0 key heads"):
        attention._arguments("decode_attention", q, k, k, table, n, None, 0, None)
