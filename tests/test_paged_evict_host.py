"""A refused eviction leaves the paged cache as it was, without a GPU."""
import pytest
import torch

import kv_reduce_b200.paged as paged
from test_paged_host import held


def filled(layers=1):
    c = paged.PagedKVCache(layers, 2, 1, 64, num_pages=30, page_size=4, device="cpu", track_weights=True)
    c.advance([21, 12])
    for i, w in enumerate(c.token_weights):
        w.copy_(torch.rand(w.shape, generator=torch.Generator().manual_seed(i)))
    return c


def test_a_refused_eviction_keeps_the_pages():
    c = filled()
    before = list(c._free), [w.clone() for w in c.token_weights]
    with pytest.raises(ValueError):          # refused by the operator: host tensors
        c.evict(8)
    held(c)
    assert (c._free, c.seq_lengths()) == (before[0], [21, 12])
    assert all(torch.equal(*x) for x in zip(c.token_weights, before[1]))


def test_a_refusal_at_a_later_layer(monkeypatch):
    c = filled(3)
    weights = [w.clone() for w in c.token_weights]
    calls = []

    def op(k, v, table, lengths, w, new_table, keep, recent, first):
        calls.append(new_table.clone())
        if len(calls) == fails_at:
            raise ValueError("refused")
        n = lengths.clamp_max(keep)
        return torch.zeros(2, keep, dtype=torch.int32), n, torch.full((2, keep), 2.0 + len(calls))

    monkeypatch.setattr(paged, "_evict_op", op)
    for fails_at in (1, 3):
        calls.clear()
        with pytest.raises(ValueError, match="refused"):
            c.evict(8)
        held(c)
        assert c.free_pages() == 30 - 9 and c.seq_lengths() == [21, 12]
        assert all(torch.equal(*x) for x in zip(c.token_weights, weights))
    fails_at = 0
    calls.clear()
    assert c.evict(8) is True
    held(c)
    assert c.free_pages() == 30 - 4 and c.seq_lengths() == [8, 8]
    assert torch.equal(calls[0], c.block_table[:, :2]) and len(calls) == 3
    for i, w in enumerate(c.token_weights):
        assert (w[:, :8] == 3.0 + i).all() and (w[:, 8:] == 0).all()


def test_eviction_looks_at_the_columns_in_use(monkeypatch):
    """A pool of more tokens than the operator takes, with short sequences."""
    c = paged.PagedKVCache(1, 2, 1, 8, num_pages=30000, page_size=16, device="cpu", track_weights=True)
    c.advance([100, 70])
    tables = []

    def op(k, v, table, lengths, w, new_table, keep, recent, first):
        tables.append(table.clone())
        return torch.zeros(2, keep, dtype=torch.int32), lengths.clamp_max(keep), torch.zeros(2, keep)

    monkeypatch.setattr(paged, "_evict_op", op)
    want = c.block_table[:, :7].clone()
    assert c.evict(40) and torch.equal(tables[0], want)
    assert c.seq_lengths() == [40, 40] and c.free_pages() == 30000 - 6
