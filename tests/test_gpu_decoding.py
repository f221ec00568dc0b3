"""Beam search over a paged cache against the same model run whole by transformers.

The two differ by the roundings of attention's 16-bit products and outputs: each
layer's output is off by a few units of 2^-11 of its size, and a log probability
by that times the logits' size.  0.05 bounds it for this model (logits of size 1,
two layers), and a wrong key, position or page moves it by far more."""
import pytest
import torch

from test_gpu_groups import _tiny_quantized_llama

pytestmark = pytest.mark.gpu


def log_probability(model, prompt, tokens, window=None, sinks=0):
    """Of `tokens` after `prompt`, with the window as an explicit mask."""
    ids = torch.tensor([prompt + tokens], device="cuda")
    n = ids.shape[1]
    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    see = j <= i
    if window:
        see &= (j > i - window) | (j < sinks)
    mask = torch.zeros(1, 1, n, n, device="cuda", dtype=model.dtype).masked_fill(~see, torch.finfo(model.dtype).min)
    logits = model(ids, attention_mask=mask).logits[0].float().log_softmax(-1)
    at = torch.arange(len(prompt) - 1, n - 1, device="cuda")
    return logits[at, ids[0, len(prompt):]]


@pytest.mark.parametrize("window,sinks", [(None, 0), (8, 2)])
@pytest.mark.parametrize("beams", [1, 3])
def test_beam_scores_are_the_models(beams, window, sinks):
    from quipsharp_b200.decoding import beam_search
    model = _tiny_quantized_llama()
    prompts = [[5, 9, 100, 3, 77, 21, 60, 8, 44, 90, 11, 12, 13, 14, 15, 16, 17], [64], [1, 2, 3]]
    tokens, scores = beam_search(model, prompts, beams, 20, window=window, sinks=sinks)
    assert tokens.shape == (3, beams, 20) and bool((scores[:, :-1] >= scores[:, 1:]).all())
    with torch.no_grad():
        for p, prompt in enumerate(prompts):
            for b in range(beams):
                want = log_probability(model, prompt, tokens[p, b].tolist(), window, sinks).sum()
                assert abs(float(want - scores[p, b])) < 0.05
            assert len({tuple(t) for t in tokens[p].tolist()}) == beams


def test_ended_beams_keep_their_score():
    from quipsharp_b200.decoding import beam_search
    model = _tiny_quantized_llama()
    prompt = [5, 9, 100, 3]
    free, _ = beam_search(model, [prompt], 1, 12)
    eos = int(free[0, 0, 5])
    tokens, scores = beam_search(model, [prompt], 1, 12, eos=eos, pad=7)
    first = free[0, 0].tolist().index(eos)
    assert tokens[0, 0].tolist() == free[0, 0, :first + 1].tolist() + [7] * (11 - first)
    with torch.no_grad():
        want = log_probability(model, prompt, tokens[0, 0, :first + 1].tolist()).sum()
    assert abs(float(want - scores[0, 0])) < 0.05


def test_prompts_in_chunks():
    """A prompt in two chunks, beside another row's, gives the logits of the whole."""
    from quipsharp_b200.decoding import PagedDecoder
    model = _tiny_quantized_llama()
    a, b = list(range(3, 40)), [90, 80, 70]
    whole = PagedDecoder(model, 3, 60).prompt([a, b], [0, 2])
    decoder = PagedDecoder(model, 3, 60)
    decoder.prompt([a[:20]], [0])
    got = decoder.prompt([a[20:], b], [0, 2])
    decoder.cache.check()
    assert decoder.cache.lengths.tolist() == [37, 0, 3]
    assert float((got - whole).float().norm() / whole.float().norm()) < 5e-3
    with pytest.raises(ValueError):
        decoder.prompt([a], [5, 1])


def test_too_few_pages_raise():
    from quipsharp_b200.decoding import beam_search
    with pytest.raises(RuntimeError, match="no free page"):
        beam_search(_tiny_quantized_llama(), [[1] * 30], 4, 20, num_pages=4)
    from quipsharp_b200.kv_cache import check_device
    check_device("cuda")
