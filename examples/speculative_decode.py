"""Speculative decoding with every part of the library: the draft model on its
packed cache, the target on its paged one, verification on the GPU.

    python examples/speculative_decode.py [--tokens 64] [--draft 4] [--temperature 0.8]

The models are small random-initialised Qwen2 (no weights to fetch); the draft
is the target with its last layer left out, so some of its tokens are accepted.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from transformers import Qwen2Config, Qwen2ForCausalLM  # noqa: E402

from kv_reduce_b200 import hf  # noqa: E402


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--draft", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=512)
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--keep", type=int, default=0, help="tokens the target's cache is brought back to (0: all)")
    a = ap.parse_args()

    def model(layers: int) -> Qwen2ForCausalLM:
        torch.manual_seed(0)
        cfg = Qwen2Config(vocab_size=2048, hidden_size=768, intermediate_size=2048, num_hidden_layers=layers,
                          num_attention_heads=6, num_key_value_heads=2, max_position_embeddings=8192,
                          attn_implementation="sdpa")
        return Qwen2ForCausalLM(cfg).to("cuda", torch.bfloat16).eval()

    target, draft = model(4), model(3)
    draft.load_state_dict(target.state_dict(), strict=False)
    hf.install_target(target)
    hf.install(draft)
    g = torch.Generator("cuda").manual_seed(1)
    prompt = torch.randint(0, 2048, (1, a.prompt), device="cuda", generator=g)
    out, rounds = hf.speculative_generate(target, draft, prompt, max_new_tokens=a.tokens, draft_tokens=a.draft,
                                          temperature=a.temperature, generator=g, keep=a.keep,
                                          recent=a.keep // 4, first=4 if a.keep else 0)
    print("new tokens:", out[0, a.prompt:].tolist())
    print(f"{len(rounds)} rounds for {a.tokens} tokens, {sum(rounds) / (len(rounds) * a.draft):.0%} of the drafted "
          "tokens accepted")


if __name__ == "__main__":
    main()
