"""Models and arguments that the paged decoder refuses (no GPU)."""
from types import SimpleNamespace

import pytest
import torch
import transformers
from transformers import AutoModelForCausalLM

from quipsharp_b200.decoding import PagedDecoder

SIZES = dict(vocab_size=120, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4,
             num_key_value_heads=2, max_position_embeddings=256, pad_token_id=0)


def tiny(name, **change):
    return AutoModelForCausalLM.from_config(getattr(transformers, name)(**{**SIZES, **change})).bfloat16()


@pytest.mark.parametrize("name,change,options,what", [
    ("Qwen3Config", dict(head_dim=16), {}, "q_norm"),
    ("Gemma2Config", dict(head_dim=16), {}, "softcapping"),
    ("GemmaConfig", dict(head_dim=16), {}, "activation"),
    ("GraniteConfig", dict(embedding_multiplier=12.0), {}, "embedding_multiplier"),
    ("GraniteConfig", dict(attention_multiplier=0.1), {}, "scores scaled"),
    ("Ernie4_5Config", dict(head_dim=16), {}, "pairing"),
    ("DiffLlamaConfig", {}, {}, "lambda"),
    ("OlmoConfig", dict(clip_qkv=8.0), {}, "clip_qkv"),
    ("LlamaConfig", dict(hidden_act="gelu"), {}, "activation"),
    ("SmolLM3Config", dict(num_hidden_layers=4), {}, "without positions"),
    ("GlmConfig", dict(head_dim=16), {}, "no gate_proj"),
    ("CohereConfig", {}, {}, "logit_scale"),
    ("MistralConfig", dict(sliding_window=32), {}, "window=32"),
    ("MistralConfig", dict(sliding_window=32), dict(window=33), "window=32"),
    ("Qwen2Config", dict(use_sliding_window=True, sliding_window=32, max_window_layers=1), {}, "window=32")])
def test_models_that_compute_something_else_are_refused(name, change, options, what):
    with pytest.raises(NotImplementedError, match=what):
        PagedDecoder(tiny(name, **change), 2, 100, **options)


@pytest.mark.parametrize("name,change,options", [
    ("LlamaConfig", {}, {}), ("LlamaConfig", dict(attention_bias=True, mlp_bias=True), dict(window=5)),
    ("MistralConfig", {}, {}), ("MistralConfig", dict(sliding_window=32), dict(window=32)),
    ("MistralConfig", dict(sliding_window=100), {}), ("Qwen2Config", dict(sliding_window=32), {}),
    ("OlmoConfig", {}, {}), ("SmolLM3Config", {}, {}), ("SeedOssConfig", dict(head_dim=16), {}), ("GraniteConfig", dict(
        attention_multiplier=0.25), {})])
def test_models_of_the_layout_are_taken(name, change, options):
    with pytest.raises(RuntimeError, match="CUDA tensors only"):  # the cache, which comes next
        PagedDecoder(tiny(name, **change), 2, 100, **options)


def bare(rows=3, vocab=10):
    """A decoder with nothing behind it: what is refused is refused before anything runs."""
    decoder = object.__new__(PagedDecoder)
    decoder.cache = SimpleNamespace(lengths=torch.zeros(rows, dtype=torch.int32))
    decoder.model = SimpleNamespace(model=SimpleNamespace(embed_tokens=torch.nn.Embedding(vocab, 8)))
    return decoder


@pytest.mark.parametrize("rows", [[-1, 0], [-2, -1], [0, 3], [1, 7]])
def test_rows_that_are_not_there_are_refused(rows):
    """Row -1 as Python counts it would take another row's prompt."""
    with pytest.raises(IndexError):
        bare().prompt([[1], [2]], rows)


@pytest.mark.parametrize("prompt", [[3, 10], [-1], [4, 1 << 40]])
def test_tokens_that_are_not_there_are_refused(prompt):
    with pytest.raises(IndexError, match="tokens from 0 to 9"):
        bare().prompt([[1], prompt], [0, 1])
