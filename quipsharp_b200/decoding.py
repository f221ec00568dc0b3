"""Generation with a quantized causal language model: the decoding operators in use.

`PagedDecoder` runs a decoder of the Llama layout (what transformers'
LlamaForCausalLM has: `model.embed_tokens`, `model.layers` with `self_attn` and
`mlp` projections, `model.rotary_emb`, `model.norm`, `lm_head`), its projections
QuantizedLinear or any module, with its keys and values in a PagedKVCache:
prompts through window_attention, further tokens through decode_attention.
`beam_search` searches over it with beam_select, forking the cache by the
parents of each step; nothing between two steps goes through the host.  The
reference leaves generation to transformers.
"""
from __future__ import annotations

import torch
from torch import Tensor, nn

from .beam import beam_select
from .kv_cache import PagedKVCache


def _rotate(x: Tensor, cos: Tensor, sin: Tensor) -> Tensor:
    """Rotary positions on x (tokens, heads, dim), cos and sin (tokens, dim), halves paired."""
    half = x.shape[-1] // 2
    turned = torch.cat((-x[..., half:], x[..., :half]), -1)
    return x * cos[:, None] + turned * sin[:, None]


class PagedDecoder:
    """A causal language model with its keys and values in pages, for `rows`
    sequences of up to `max_len` tokens.

    window and sinks: every token sees the last `window` tokens (None: all) and
    the first `sinks`.  num_pages defaults to what all rows can fill."""

    def __init__(self, model: nn.Module, rows: int, max_len: int, num_pages: int | None = None, page_size: int = 16,
                 window: int | None = None, sinks: int = 0):
        self.model, self.window, self.sinks = model, window, sinks
        self.layers = model.model.layers
        config, weight = model.config, model.model.embed_tokens.weight
        self.heads = config.num_attention_heads
        self.kv_heads = getattr(config, "num_key_value_heads", None) or self.heads
        self.dim = getattr(config, "head_dim", None) or config.hidden_size // self.heads
        if num_pages is None:
            num_pages = rows * (-(-max_len // page_size) + 1)
        self.cache = PagedKVCache(len(self.layers), self.kv_heads, self.dim, num_pages, rows, max_len, page_size,
                                  weight.dtype, weight.device)

    def _forward(self, ids: Tensor, positions: Tensor, cu: Tensor | None) -> Tensor:
        """The last hidden states of packed tokens whose places the cache already counts."""
        x = self.model.model.embed_tokens(ids)
        cos, sin = self.model.model.rotary_emb(x[None], positions[None])
        cos, sin = cos[0], sin[0]
        seen = dict(window=self.window, sinks=self.sinks)
        for i, layer in enumerate(self.layers):
            h, attn = layer.input_layernorm(x), layer.self_attn
            q = _rotate(attn.q_proj(h).view(-1, self.heads, self.dim), cos, sin)
            k = _rotate(attn.k_proj(h).view(-1, self.kv_heads, self.dim), cos, sin)
            self.cache.write(i, k, attn.v_proj(h).view(-1, self.kv_heads, self.dim), cu)
            o = self.cache.decode(i, q, **seen) if cu is None else self.cache.window(i, q, cu, **seen)
            x = x + attn.o_proj(o.flatten(1))
            h, mlp = layer.post_attention_layernorm(x), layer.mlp
            x = x + mlp.down_proj(nn.functional.silu(mlp.gate_proj(h)) * mlp.up_proj(h))
        return self.model.model.norm(x)

    @torch.no_grad()
    def prompt(self, prompts: list[list[int]], rows: list[int]) -> Tensor:
        """Appends one prompt (or a chunk of one) to each of the given rows, whose
        order is ascending; returns the logits after each one's last token."""
        if list(rows) != sorted(set(rows)) or len(rows) != len(prompts) or not all(prompts):
            raise ValueError("prompts must not be empty and their rows ascending, one for each")
        device = self.cache.lengths.device
        new = [0] * len(self.cache.lengths)
        for r, p in zip(rows, prompts):
            new[r] = len(p)
        counts = torch.tensor(new, dtype=torch.int32)
        cu = torch.cat((counts.new_zeros(1), counts.cumsum(0, dtype=torch.int32)))
        row = torch.repeat_interleave(torch.arange(len(new)), counts.long()).to(device)
        new, cu = counts.to(device), cu.to(device)
        before = self.cache.lengths.clone()
        self.cache.extend(new)
        ids = torch.tensor([t for p in prompts for t in p], device=device)
        positions = before[row] + torch.arange(len(ids), device=device) - cu[row]
        x = self._forward(ids, positions, cu)
        last = (cu[1:] - 1)[torch.tensor(rows, device=device)].long()
        return self.model.lm_head(x[last])

    @torch.no_grad()
    def step(self, ids: Tensor) -> Tensor:
        """Appends one token to every row; returns the logits after it (rows, vocabulary)."""
        self.cache.extend(1)
        return self.model.lm_head(self._forward(ids, self.cache.lengths - 1, None))


@torch.no_grad()
def beam_search(model: nn.Module, prompts: list[list[int]], beams: int, new_tokens: int, eos: int | None = None,
                pad: int = 0, **options):
    """The `beams` likeliest continuations of each prompt by up to `new_tokens`
    tokens, found by beam search: (tokens (prompts, beams, new_tokens), log
    probabilities (prompts, beams)), best first.  A beam ends with `eos`; what
    follows it is `pad`.  options: see PagedDecoder."""
    if beams < 1 or new_tokens < 1:
        raise ValueError("beams and new_tokens must be positive")
    batch, longest = len(prompts), max(map(len, prompts))
    decoder = PagedDecoder(model, batch * beams, longest + new_tokens, **options)
    first = torch.arange(0, batch * beams, beams, dtype=torch.int32, device=decoder.cache.lengths.device)
    # the first step: one live beam of each prompt, its logits shared by all
    logits = decoder.prompt(prompts, list(range(0, batch * beams, beams)))[:, None].expand(-1, beams, -1)
    scores = torch.full((batch, beams), float("-inf"), device=logits.device)
    scores[:, 0] = 0.0
    ended = torch.zeros(batch, beams, dtype=torch.bool, device=logits.device)
    history = []
    for i in range(new_tokens):
        scores, parents, tokens = beam_select(logits, scores, beams, ended if eos is not None else None, pad)
        history.append((parents, tokens))
        if eos is not None:
            ended = ended.gather(1, parents.long()) | (tokens == eos)
        if i + 1 == new_tokens:
            break
        decoder.cache.fork((parents + first[:, None]).flatten())
        logits = decoder.step(tokens.flatten()).view(batch, beams, -1)
    out, at = [], torch.arange(beams, device=logits.device).expand(batch, -1)
    for parents, tokens in reversed(history):
        out.append(tokens.gather(1, at))
        at = parents.long().gather(1, at)
    decoder.cache.check()
    return torch.stack(out[::-1], -1), scores
