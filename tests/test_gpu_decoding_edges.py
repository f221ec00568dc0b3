"""Beam search over a paged cache: arguments at their edges."""
import pytest
import torch

from test_gpu_groups import _tiny_quantized_llama

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pad", [-100, 1 << 20])
def test_pad_need_not_be_a_token(pad):
    """What follows an ended beam is only written down: the model never sees it."""
    from quipsharp_b200.decoding import beam_search
    model = _tiny_quantized_llama()
    prompts = [[5, 9, 100, 3], [64]]
    free, _ = beam_search(model, prompts, 3, 10)
    eos = int(free[0, 0, 4])
    want, scores = beam_search(model, prompts, 3, 10, eos=eos, pad=7)
    got, same = beam_search(model, prompts, 3, 10, eos=eos, pad=pad)
    after = (want == eos).cumsum(-1) - (want == eos).int() > 0
    assert after.any() and torch.equal(got, want.masked_fill(after, pad)) and torch.equal(same, scores)
