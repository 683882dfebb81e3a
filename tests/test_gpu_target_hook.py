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
