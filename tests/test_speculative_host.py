"""The generation loop's host side, with models and operators that are fakes."""
from types import SimpleNamespace

import pytest
import torch

pytest.importorskip("transformers")
from kv_reduce_b200 import hf  # noqa: E402
from kv_reduce_b200.speculative import VerifyResult  # noqa: E402


class Model:
    """Logits that prefer token 3; refuses ids that no embedding has."""

    def __init__(self, vocab=8):
        self.config = SimpleNamespace(head_dim=64, num_hidden_layers=1, num_key_value_heads=1)
        self.model = SimpleNamespace(layers=[None])
        self.device, self.dtype, self.vocab, self.seen = torch.device("cpu"), torch.bfloat16, vocab, []

    def __call__(self, ids, past_key_values=None, use_cache=True, position_ids=None):
        self.seen += ids.flatten().tolist()
        assert min(self.seen) >= 0 and max(self.seen) < self.vocab
        past_key_values.grow(ids.shape[1])
        return SimpleNamespace(logits=torch.eye(self.vocab)[3].expand(1, ids.shape[1], -1))


class DraftCache:
    def __init__(self):
        self.n = 0

    def grow(self, n):
        self.n += n

    def get_seq_length(self):
        return self.n

    def crop(self, n):
        self.n = n

    def commit(self):
        pass


@pytest.fixture
def models(monkeypatch):
    monkeypatch.setattr(hf.PackedDraftCache, "empty", classmethod(lambda cls, *a, **kw: DraftCache()))
    monkeypatch.setattr(hf.PagedTargetCache, "grow", lambda self, n: self.pages.advance(n), raising=False)
    return Model(), Model()


def answers(monkeypatch, rows):
    rows = iter(rows)

    def verify(target, draft, tokens, *a, **kw):
        accepted, row = next(rows)
        return VerifyResult(torch.tensor([row]), torch.tensor([accepted], dtype=torch.int32), torch.zeros(1, 2))

    monkeypatch.setattr(hf, "verify_draft_tokens", verify)


def test_generation(models, monkeypatch):
    answers(monkeypatch, [(2, [3, 3, 5]), (0, [4, -1, -1]), (1, [3, 6, -1])])
    out, rounds = hf.speculative_generate(*models, torch.tensor([[1, 2]]), max_new_tokens=7, draft_tokens=2)
    assert out.tolist() == [[1, 2, 3, 3, 3, 5, 4, 3, 6]] and rounds == [2, 0, 1]


@pytest.mark.parametrize("accepted,row", [(0, [-1, -1, -1]), (1, [3, -1, -1]), (2, [3, 3, -1])])
def test_logits_without_any_weight_end_the_generation(models, monkeypatch, accepted, row):
    """A target row of NaN gives token -1, which no embedding has: an error on
    the host, before a model sees it."""
    answers(monkeypatch, [(2, [3, 3, 5]), (accepted, row), (2, [3, 3, 5])])
    with pytest.raises(RuntimeError, match="logits"):
        hf.speculative_generate(*models, torch.tensor([[1, 2]]), max_new_tokens=20, draft_tokens=2)
    assert min(models[0].seen + models[1].seen) >= 0
