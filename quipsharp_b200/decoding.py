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

import sys

import torch
from torch import Tensor, nn

from .beam import beam_select
from .kv_cache import PagedKVCache


def _rotate(x: Tensor, cos: Tensor, sin: Tensor) -> Tensor:
    """Rotary positions on x (tokens, heads, dim), cos and sin (tokens, dim), halves paired."""
    half = x.shape[-1] // 2
    turned = torch.cat((-x[..., half:], x[..., :half]), -1)
    return x * cos[:, None] + turned * sin[:, None]


_PARTS = {"self_attn": ("q_proj", "k_proj", "v_proj", "o_proj"), "mlp": ("gate_proj", "up_proj", "down_proj")}
# settings of a configuration under which a model of these names computes something else
_SETTINGS = {"embedding_multiplier": 1, "residual_multiplier": 1, "logits_scaling": 1, "logit_scale": 1, "clip_qkv": None,
             "attn_logit_softcapping": None, "final_logit_softcapping": None}


def _refuse_other_models(model: nn.Module, dim: int, max_len: int, window: int | None) -> None:
    """NotImplementedError for a model that has the Llama layout's names but more in it, or
    something else behind them, so that PagedDecoder's outputs would not be the model's."""
    def refuse(what):
        raise NotImplementedError(f"PagedDecoder runs the Llama layout; this model has {what}")

    config, inner = model.config, model.model
    for name, plain in _SETTINGS.items():
        if getattr(config, name, plain) not in (plain, None):
            refuse(f"{name} = {getattr(config, name)}")
    rope = getattr(config, "rope_parameters", None) or {}
    if rope.get("llama_4_scaling_beta") and max_len > rope.get("original_max_position_embeddings", 0):
        refuse("queries scaled by their position")
    kinds, own = getattr(config, "layer_types", None), getattr(config, "sliding_window", None)
    if set(kinds or ()) - {"full_attention", "sliding_attention"}:
        refuse(f"layers of the types {sorted(set(kinds))}")
    slides = "sliding_attention" in kinds if kinds else getattr(config, "use_sliding_window", True)
    if own and slides and max_len > own and (window is None or window > own):
        refuse(f"a sliding window of {own} tokens, less than max_len = {max_len}: give window={own}, or less")

    weight = inner.embed_tokens.weight
    acts = {}
    for layer in inner.layers:
        for module, names in ((layer, ("input_layernorm", "post_attention_layernorm", *_PARTS)),
                              *((getattr(layer, part, None), names) for part, names in _PARTS.items())):
            gone = [n for n in names if not hasattr(module, n)]
            if gone:
                refuse(f"no {', '.join(gone)}")
            more = [n for n, _ in module.named_parameters(recurse=False)]
            more += [n for n, m in module.named_children() if n not in names and any(True for _ in m.parameters())]
            if more:
                refuse(f"{', '.join(more)} in {type(module).__name__}")
        attn, act = layer.self_attn, getattr(layer.mlp, "act_fn", None)
        scaling = getattr(attn, "scaling", None)
        if isinstance(scaling, (int, float)) and abs(scaling * dim ** 0.5 - 1) > 1e-6:
            refuse(f"scores scaled by {scaling}")
        if not getattr(attn, "use_rope", True):
            refuse("layers without positions")
        if callable(act):
            acts[type(act)] = act
    x = torch.linspace(-4, 4, 2 * dim, device=weight.device).view(1, 2, 1, dim)  # two heads of a token
    for act in acts.values():
        if not torch.allclose(act(x), nn.functional.silu(x), atol=1e-5):
            refuse(f"the activation {act}")
    cos, sin = inner.rotary_emb(x.new_zeros(1, 1, weight.shape[1]), torch.tensor([[5]], device=weight.device))
    if cos.shape[-1] != dim:
        refuse("positions on a part of a head's dimensions")
    turn = getattr(sys.modules.get(type(attn).__module__), "apply_rotary_pos_emb", None)
    if turn is None:
        return
    try:
        turned = turn(x, x, cos, sin)[0]
    except TypeError:  # called in another way: nothing to compare
        return
    if not torch.allclose(turned, _rotate(x.transpose(1, 2)[0], cos[0], sin[0])[:, :, None], atol=1e-5):
        refuse("another pairing of dimensions in its rotary positions")


class PagedDecoder:
    """A causal language model with its keys and values in pages, for `rows`
    sequences of up to `max_len` tokens.

    window and sinks: every token sees the last `window` tokens (None: all) and
    the first `sinks`.  num_pages defaults to what all rows can fill.  Models that
    have the Llama layout's names but compute something else (norms of queries and
    keys, other scales, activations or positions, a shorter window of their own)
    are refused."""

    def __init__(self, model: nn.Module, rows: int, max_len: int, num_pages: int | None = None, page_size: int = 16,
                 window: int | None = None, sinks: int = 0):
        self.model, self.window, self.sinks = model, window, sinks
        self.layers = model.model.layers
        config, weight = model.config, model.model.embed_tokens.weight
        self.heads = config.num_attention_heads
        self.kv_heads = getattr(config, "num_key_value_heads", None) or self.heads
        self.dim = getattr(config, "head_dim", None) or config.hidden_size // self.heads
        _refuse_other_models(model, self.dim, max_len, window)
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
        if rows and not 0 <= rows[0] <= rows[-1] < len(new):
            raise IndexError(f"rows go from 0 to {len(new) - 1}, got {list(rows)}")
        vocab = self.model.model.embed_tokens.weight.shape[0]
        if not all(0 <= t < vocab for p in prompts for t in p):  # the embedding would stop the device
            raise IndexError(f"prompts hold tokens from 0 to {vocab - 1}")
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
            tokens = tokens.masked_fill(ended, 0)  # nothing reads their logits, and `pad` need not be a token
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
