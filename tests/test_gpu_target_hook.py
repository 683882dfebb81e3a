"""The target's hook over prompts of different lengths."""
import pytest
import torch

from test_gpu_speculative import tiny_qwen2

pytestmark = pytest.mark.gpu


@torch.inference_mode()
def test_prompts_padded_on_the_right(built_lib):
    """Padding on the right and a crop: each sequence as the model alone."""
    from kv_reduce_b200 import hf

    model = tiny_qwen2(8)
    g = torch.Generator("cuda").manual_seed(9)
    lengths = [90, 61, 17]
    ids = torch.randint(0, 512, (3, 96), device="cuda", generator=g)
    want = [model(ids[b:b + 1, :n + 4]).logits[0, n:].float() for b, n in enumerate(lengths)]
    hf.install_target(model)
    held = torch.tensor(lengths, device="cuda")[:, None]
    mask = (torch.arange(90, device="cuda") < held).long()
    for m in (mask, None):
        cache = hf.PagedTargetCache.for_model(model, 3, max_tokens=128)
        model(ids[:, :90], attention_mask=m, past_key_values=cache, use_cache=True)
        cache.crop(lengths)
        step = torch.stack([ids[b, n:n + 4] for b, n in enumerate(lengths)])
        got = model(step, past_key_values=cache, use_cache=True, position_ids=held + torch.arange(4, device="cuda")).logits
        for b in range(3):
            assert torch.nn.functional.cosine_similarity(got[b].float(), want[b], dim=-1).min().item() > 0.995
    with pytest.raises(ValueError, match="right"):
        model(ids[:, :90], attention_mask=mask.flip(1), use_cache=True,
              past_key_values=hf.PagedTargetCache.for_model(model, 3, max_tokens=128))


@torch.inference_mode()
def test_sliding_layers(built_lib):
    """A model with a sliding layer: its own logits, past the window."""
    transformers = pytest.importorskip("transformers")
    from kv_reduce_b200 import hf

    torch.manual_seed(3)
    cfg = transformers.Qwen2Config(vocab_size=512, hidden_size=768, intermediate_size=1024, num_hidden_layers=2,
                                   num_attention_heads=6, num_key_value_heads=2, use_sliding_window=True,
                                   sliding_window=24, max_window_layers=1, attn_implementation="sdpa")
    model = transformers.Qwen2ForCausalLM(cfg).to(device="cuda", dtype=torch.bfloat16).eval()
    for x in model.model.layers:                     # (attention that counts: the output's weights are small at random)
        x.self_attn.v_proj.weight.mul_(8)
    ids = torch.randint(0, 512, (1, 150), device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    want = model(ids).logits.float()
    hf.install_target(model)
    cache = hf.PagedTargetCache.for_model(model, 1, max_tokens=160)
    got = [model(ids[:, a:b], past_key_values=cache, use_cache=True).logits
           for a, b in ((0, 100), (100, 101), (101, 109), (109, 150))]
    cos = torch.nn.functional.cosine_similarity(torch.cat(got, 1).float(), want, dim=-1)
    assert cos.min().item() > 0.995
