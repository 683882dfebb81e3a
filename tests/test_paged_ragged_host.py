"""What the paged cache hands to the append after unequal advances, without a GPU."""
import pytest
import torch

import kv_reduce_b200.paged as paged


@pytest.fixture
def calls(monkeypatch):
    got = []
    monkeypatch.setattr(paged, "_append_op", lambda *a: got.append(("append", a[-1])))
    monkeypatch.setattr(paged, "_attention_op", lambda *a: (got.append(("attention", a[-1])), a[0])[1:] * 2)
    monkeypatch.setattr(paged, "_evict_op", None)
    return got


def test_counts_follow_the_advances(calls):
    c = paged.PagedKVCache(1, 3, 1, 64, num_pages=40, page_size=8, device="cpu")

    def step(T):
        x = torch.zeros(3, 1, T, 64, dtype=torch.bfloat16)
        c.append(0, x, x)
        c.attention(0, x)
        return [None if n is None else n.tolist() for _, n in calls[-2:]]

    c.advance(7)
    assert step(7) == [None, None]
    c.advance([1, 5, 0])
    assert step(5) == [[1, 5, 0], [1, 5, 0]]
    with pytest.raises(ValueError):           # rows that advance made no room for
        c.append(0, torch.zeros(3, 1, 6, 64), torch.zeros(3, 1, 6, 64))
    assert step(1) == [[1, 5, 0], [1, 5, 0]]
    c.advance([2, 2, 2])
    assert step(2) == [None, None]
    c.advance(4)
    c.crop([n - x for n, x in zip(c.seq_lengths(), (4, 1, 3))])
    assert step(3) == [[0, 3, 1], None]       # what is left of the four; the queries stay the newest of every sequence
    c.advance(2)
    c.advance([3, 3, 0])                      # two advances, one append
    assert step(5) == [[5, 5, 2], [5, 5, 2]]
    c.advance(1)
    c.advance(3)
    assert step(4) == [None, None] and step(2) == [None, None]
    c.crop(0)
    with pytest.raises(ValueError):
        c.append(0, torch.zeros(3, 1, 1, 64), torch.zeros(3, 1, 1, 64))
