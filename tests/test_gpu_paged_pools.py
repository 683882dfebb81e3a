"""Caches whose pool, and so whose block table, is far wider than a sequence."""
import math

import pytest
import torch

from test_gpu_paged import kvr, make, reference  # noqa: F401  (kvr: the fixture)

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


def peak(call):
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = call()
    torch.cuda.synchronize()
    return got, torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("B,HQ,H,D,T,width", [(32, 32, 8, 64, 5, 12000), (5, 12, 2, 128, 9, 100000),
                                              (7, 32, 8, 64, 1, 200000), (2, 16, 1, 128, 16, 140000)])
def test_scores_of_a_part_of_the_batch(kvr, B, HQ, H, D, T, width):  # noqa: F811
    """Token weights in wide tables: 2 GiB of scores at a time, or one
    sequence's; rows of unequal tables, counts and weights with row strides."""
    lengths = [(i * 397) % 900 + 3 for i in range(B)]
    q, k, v, table, n = make(lengths, HQ, H, D, T, 16, seed=B, max_pages=width)
    w = torch.full((B, width * 16 + 4), 0.25, device="cuda")
    counts = torch.tensor([1 + i % T for i in range(B)], dtype=torch.int32, device="cuda")
    for new in (None, counts):
        w.fill_(0.25)
        (out, lse), used = peak(lambda: kvr.paged_decode_attention(q, k, v, table, n, token_weights=w, return_lse=True,
                                                                   new_counts=new))
        one = HQ * T * width * 16 * 4
        assert used <= max(2 << 30, one) + (64 << 20) and B * one > 2 << 30
        for b in range(B):
            at, m = slice(b, b + 1), T if new is None else int(new[b])
            want, size, want_lse, want_w = reference(q[at, :, T - m:], k, v, table[at], n[at])
            assert ((out[at, :, T - m:].double() - want).abs() <= (2 ** -8 + 2 ** -12) * size + 1e-7).all()
            assert (out[b, :, :T - m] == 0).all()
            empty = want_lse == -math.inf
            assert ((lse[at, :, T - m:].double() - want_lse)[~empty].abs() <= 2 ** -14).all()
            got = w[at, :want_w.shape[1]].double() - 0.25
            assert ((got - want_w).abs() <= 2 ** -14 * want_w + 1e-6).all()
            assert (w[b, want_w.shape[1]:] == 0.25).all()


def test_weights_of_a_cache_with_a_wide_pool(kvr):  # noqa: F811
    """The class's table is as wide as its pool; the scores go by the sequences."""
    cache = kvr.PagedKVCache(1, 8, 1, 64, num_pages=60000, page_size=8, track_weights=True)
    g = torch.Generator(device="cuda").manual_seed(2)
    cache.advance(200)
    k, v, q = (torch.randn(8, h, 200, 64, device="cuda", generator=g).to(torch.bfloat16) for h in (1, 1, 4))
    cache.append(0, k, v)
    out, used = peak(lambda: cache.attention(0, q[:, :, -2:].contiguous()))
    assert used <= 32 << 20
    want, size, _, want_w = reference(q[:, :, -2:], cache.key_pages[0], cache.value_pages[0], cache.block_table[:, :25],
                                      cache.lengths)
    assert ((out.double() - want).abs() <= (2 ** -8 + 2 ** -12) * size + 1e-7).all()
    got = cache.token_weights[0]
    assert ((got[:, :200].double() - want_w).abs() <= 2 ** -14 * want_w + 1e-6).all() and (got[:, 200:] == 0).all()
