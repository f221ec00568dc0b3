"""Beam search with a small quantized Llama of random weights: every projection is a
3-bit QuantizedLinear, keys and values live in a paged cache under a sliding window whose
first tokens stay visible.

    python examples/beam_search.py [beams] [new tokens]

With a real checkpoint, replace `tiny_model()` by
`quipsharp_b200.checkpoint.load_quantized_checkpoint(path, device="cuda")`."""
import os
import sys

import torch
from transformers import LlamaConfig, LlamaForCausalLM

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from quipsharp_b200 import synthetic as syn  # noqa: E402
from quipsharp_b200.checkpoint import QuantizedLinear  # noqa: E402
from quipsharp_b200.codebooks import E8OneBitCodebook, E8PCodebook  # noqa: E402
from quipsharp_b200.decoding import beam_search  # noqa: E402
from quipsharp_b200.groups import fuse_linear_groups  # noqa: E402
from quipsharp_b200.quantize import RVQCodebookAdapter  # noqa: E402
from quipsharp_b200.rvq import RVQStage  # noqa: E402


def quantized(out_features: int, in_features: int, seed: int) -> QuantizedLinear:
    lay = syn.make_layer(out_features, in_features, (syn.E8P, syn.E8_1BIT), seed=seed, layer_scale=0.5 / in_features ** 0.5)
    mod = QuantizedLinear(in_features, out_features, 8, lay.transform_kind, num_stages=2)
    with torch.no_grad():
        mod.codes.copy_(lay.codes)
        mod.scale.copy_(torch.tensor(lay.layer_scale))
        for name in ("su", "sv") if lay.transform_kind == "rht" else ("phase_u", "phase_v"):
            getattr(mod, name).copy_(getattr(lay, name))
    mod.codebook = RVQCodebookAdapter([RVQStage(E8PCodebook(), lay.stage_scales[0]),
                                       RVQStage(E8OneBitCodebook(), lay.stage_scales[1])])
    return mod


def tiny_model(dtype=torch.bfloat16, device="cuda"):
    torch.manual_seed(0)
    config = LlamaConfig(vocab_size=1000, hidden_size=512, intermediate_size=1408, num_hidden_layers=4,
                         num_attention_heads=8, num_key_value_heads=2, max_position_embeddings=2048)
    model = LlamaForCausalLM(config).to(dtype)
    for i, (name, mod) in enumerate(list(model.named_modules())):
        if isinstance(mod, torch.nn.Linear) and ".layers." in name:
            parent, _, attr = name.rpartition(".")
            setattr(model.get_submodule(parent), attr, quantized(mod.out_features, mod.in_features, seed=i))
    model = model.to(device).eval()
    fuse_linear_groups(model)
    return model


def main() -> None:
    beams, new_tokens = (int(a) for a in (sys.argv[1:] + ["4", "24"][len(sys.argv) - 1:])[:2])
    prompts = [torch.randint(0, 1000, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (70, 9, 131)]
    tokens, scores = beam_search(tiny_model(), prompts, beams, new_tokens, window=64, sinks=4)
    for p, (t, s) in enumerate(zip(tokens.tolist(), scores.tolist())):
        for b in range(beams):
            print(f"prompt {p} beam {b} log probability {s[b]:8.3f}: {t[b]}")


if __name__ == "__main__":
    main()
