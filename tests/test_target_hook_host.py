"""The target's hook on a small Qwen2 model without a GPU (the operators are fakes)."""
import pytest
import torch

transformers = pytest.importorskip("transformers")
import kv_reduce_b200.paged as paged  # noqa: E402
from kv_reduce_b200 import hf  # noqa: E402


def tiny(attn="sdpa", **kw):
    torch.manual_seed(0)
    cfg = transformers.Qwen2Config(vocab_size=64, hidden_size=128, intermediate_size=64, num_hidden_layers=2,
                                   num_attention_heads=2, num_key_value_heads=1, attn_implementation=attn, **kw)
    return transformers.Qwen2ForCausalLM(cfg).to(torch.bfloat16).eval()


@pytest.fixture
def calls(monkeypatch):
    got = []
    monkeypatch.setattr(paged, "_append_op", lambda *a: None)

    def attention(q, k, v, table, lengths, scale, window, sinks, *a):
        got.append((window, sinks))
        return torch.zeros_like(q), None

    monkeypatch.setattr(paged, "_attention_op", attention)
    return got


@torch.inference_mode()
@pytest.mark.parametrize("attn", ["sdpa", "eager"])
def test_left_padding_is_refused(calls, attn):
    model = tiny(attn)
    hf.install_target(model)
    ids = torch.arange(12).view(2, 6)
    left = torch.tensor([[1] * 6, [0, 0, 1, 1, 1, 1]])
    cache = hf.PagedTargetCache.for_model(model, 2, max_tokens=32)
    with pytest.raises(ValueError, match="right"):
        model(ids, attention_mask=left, past_key_values=cache, use_cache=True)
    assert cache.pages.seq_lengths() == [0, 0]           # and nothing was taken in
    for mask in (left.flip(1), torch.ones_like(left), None):
        cache = hf.PagedTargetCache.for_model(model, 2, max_tokens=32)
        model(ids, attention_mask=mask, past_key_values=cache, use_cache=True)
        assert cache.pages.seq_lengths() == [6, 6]
        cache.crop([6, 4])
        model(ids[:, :1], past_key_values=cache, use_cache=True, position_ids=torch.tensor([[6], [4]]))
        assert cache.pages.seq_lengths() == [7, 5] and len(calls) == 2
        calls.clear()


@torch.inference_mode()
def test_sliding_layers_keep_their_window(calls):
    """A layer with a window of its own is given it; the cache's may be tighter."""
    model = tiny(use_sliding_window=True, sliding_window=10, max_window_layers=1)
    assert [x.self_attn.sliding_window for x in model.model.layers] == [None, 10]
    hf.install_target(model)
    ids = torch.arange(6)[None]
    for kw, want in ((dict(), [(0, 0), (10, 0)]), (dict(window=7, sinks=2), [(7, 2), (7, 2)]),
                     (dict(window=20, sinks=2), [(20, 2), (10, 0)])):
        cache = hf.PagedTargetCache.for_model(model, 1, max_tokens=32, **kw)
        for _ in range(2):
            model(ids, past_key_values=cache, use_cache=True)
        assert calls == want
        calls.clear()
