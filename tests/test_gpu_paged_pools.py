"""Caches whose pool, and so whose block table, is far wider than a sequence."""
import pytest
import torch

from test_gpu_paged import kvr  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


def test_eviction_in_a_pool_of_more_tokens_than_a_table_may_have(kvr):  # noqa: F811
    H, D, page = 1, 64, 16
    cache = kvr.PagedKVCache(1, 3, H, D, num_pages=21000, page_size=page, track_weights=True)
    assert cache.max_pages * page > 320000
    g = torch.Generator(device="cuda").manual_seed(0)
    lengths, keep, recent, first = [500, 90, 1000], 120, 30, 2
    cache.advance(lengths)
    k, v = (torch.randn(3, H, 1000, D, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    cache.append(0, k, v)
    cache.token_weights[0].copy_(torch.rand(cache.token_weights[0].shape, device="cuda", generator=g))
    w = cache.token_weights[0].clone()
    assert cache.evict(keep, recent=recent, first=first)
    assert cache.seq_lengths() == [120, 90, 120]
    for b, n in enumerate(lengths):
        x = w[b, :n].clone()
        if n > keep:
            x[:first] = x[n - recent:] = 2
        kept = x.topk(min(n, keep)).indices.sort().values
        assert torch.equal(cache.token_weights[0][b, :len(kept)], w[b][kept])
        j = torch.arange(len(kept), device="cuda")
        at = cache.block_table[b].long()[j // page], slice(None), j % page
        assert torch.equal(cache.key_pages[0][at], k[b, :, 1000 - n + kept].transpose(0, 1))
        assert torch.equal(cache.value_pages[0][at], v[b, :, 1000 - n + kept].transpose(0, 1))
