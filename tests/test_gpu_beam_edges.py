"""beam_select at the edges of what logits and arguments may be (see test_gpu_beam for the
plain form and the tolerance)."""
import pytest
import torch

from quipsharp_b200.beam import beam_select
from test_gpu_beam import check, spread

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks_of_the_types_lowest_value(dtype):
    """Vocabularies masked with the type's lowest number, whose product with log2(e) is past
    float32's range: pieces and whole rows of it, and its largest number too."""
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x, s = spread(3, 4, 20001, dtype, 9)
    x[0, :, 1000:] = low         # one live stretch
    x[0, 1, :15000] = low        # none in that row
    x[0, 2, 7::2] = low          # every other one
    x[1, 0] = low                # a row of nothing else
    x[1, 1] = low
    x[1, 1, 19000:19020] = torch.arange(20, device=DEV, dtype=dtype)
    x[1, 2, 5:] = -float("inf")
    x[1, 2, :5] = low
    x[2, 0, 4321] = high         # takes the whole probability
    x[2, 1, :] = low / 2
    x[2, 1, ::2] = low           # nothing beside the others
    check(x, s, 12)
    check(x[:, :1], s[:, :1], 4)
    check(x[1:2, 1:3], s[1:2, 1:3], 20)
