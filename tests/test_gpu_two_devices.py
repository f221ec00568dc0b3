"""The decoding operators on a second device of one process."""
import pytest
import torch

from quipsharp_b200 import attention as at
from quipsharp_b200 import kv_cache as kc
from quipsharp_b200.beam import beam_select

pytestmark = pytest.mark.gpu


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_every_operator_on_each_device():
    """What asks for more than 48 KB of shared memory runs on each device, the current one or not."""
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(400, 2, 16, 128, generator=g).half() for _ in range(2))
    q = torch.randn(6, 8, 128, generator=g).half()
    table = torch.randperm(400, generator=g).int().view(2, 200)
    lengths, cu = torch.tensor([3000, 900], dtype=torch.int32), torch.tensor([0, 4, 6], dtype=torch.int32)
    logits, scores = torch.randn(1, 64, 9000, generator=g), torch.zeros(1, 64)
    counts = torch.zeros(20000, dtype=torch.int32)
    outs = []
    for dev in ("cuda:0", "cuda:1"):
        a = [t.to(dev) for t in (q, k, v, table, lengths)]
        outs.append([at.decode_attention(a[0][:2], *a[1:]), at.window_attention(*a, cu.to(dev)),
                     *beam_select(logits.to(dev), scores.to(dev), 64),
                     *kc.extend_pages(a[3], a[4], counts.to(dev), lengths.to(dev) // 30, 16)])
        torch.cuda.synchronize(dev)
    for x, y in zip(*outs):
        assert torch.equal(x.cpu(), y.cpu())
