"""Sequences with different numbers of new tokens in one step.  Tolerances as
derived in test_gpu_paged.py."""
import math

import pytest
import torch

from test_gpu_paged import kvr, make, reference  # noqa: F401  (kvr: the fixture)

pytestmark = pytest.mark.gpu


def test_append_after_a_ragged_advance(kvr):  # noqa: F811
    """Only the rows that advance made room for are written."""
    H, D = 2, 64
    cache = kvr.PagedKVCache(1, 4, H, D, num_pages=40, page_size=8)
    g = torch.Generator(device="cuda").manual_seed(0)
    held = [torch.zeros(0, H, D, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    for more in (12, [1, 5, 0, 3], [0, 0, 2, 0], 2, [4, 4, 4, 1]):
        cache.advance(more)
        more = [more] * 4 if isinstance(more, int) else more
        T = max(more)
        k = torch.randn(4, H, T, D, device="cuda", generator=g).to(torch.bfloat16)
        cache.append(0, k, -k)
        for b, m in enumerate(more):
            held[b] = torch.cat([held[b], k[b, :, T - m:].transpose(0, 1)])
            j = torch.arange(len(held[b]), device="cuda")
            assert cache.seq_lengths()[b] == len(held[b])
            pages = cache.block_table[b].long()[j // 8]
            assert torch.equal(cache.key_pages[0][pages, :, j % 8], held[b])
            assert torch.equal(cache.value_pages[0][pages, :, j % 8], -held[b])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("HQ,H,D,window,sinks", [(12, 2, 128, 0, 0), (8, 2, 64, 70, 3), (16, 1, 128, 300, 0)])
def test_attention_with_counts(kvr, HQ, H, D, window, sinks, dtype):  # noqa: F811
    """Every sequence as if it came alone with its own number of queries,
    whatever the padding holds; padding gives zeros and adds no weight."""
    lengths = [300, 7, 1029, 3, 128, 0, 2000, 64]
    counts = [5, 1, 0, 5, 3, 2, 4, 9]
    T = 5
    q, k, v, table, n = make(lengths, HQ, H, D, T, 16, dtype, seed=window)
    for b, m in enumerate(counts):
        q[b, :, :max(0, T - m)] = (math.nan, 1e4, math.inf)[b % 3]
    w = torch.full((len(lengths), table.shape[1] * 16), 0.25, device="cuda")
    out, lse = kvr.paged_decode_attention(q, k, v, table, n, window=window, sinks=sinks, token_weights=w,
                                          return_lse=True, new_counts=torch.tensor(counts, dtype=torch.int32).cuda())
    u = 2.0 ** -9 if dtype == "bf16" else 2.0 ** -12
    for b, m in enumerate(counts):
        m = min(m, T)
        assert (out[b, :, :T - m] == 0).all() and (lse[b, :, :T - m] == -math.inf).all()
        one = slice(b, b + 1)
        if m == 0:
            assert (w[b] == 0.25).all()
            continue
        want, size, want_lse, want_w = reference(q[one, :, T - m:], k, v, table[one], n[one], window, sinks)
        assert ((out[one, :, T - m:].double() - want).abs() <= (2 * u + 2 ** -12) * size + 1e-7).all()
        empty = want_lse == -math.inf
        got = lse[one, :, T - m:].double()
        assert torch.equal(got == -math.inf, empty) and ((got - want_lse)[~empty].abs() <= 2 ** -14).all()
        assert ((w[one].double() - 0.25 - want_w).abs() <= 2 ** -14 * want_w + 1e-6).all()
    full = kvr.paged_decode_attention(q, k, v, table, n, window=window, sinks=sinks,
                                      new_counts=torch.full((8,), T, dtype=torch.int32, device="cuda"))
    same = kvr.paged_decode_attention(q, k, v, table, n, window=window, sinks=sinks)
    assert torch.equal(full.view(torch.int16), same.view(torch.int16))


def test_cache_attention_after_a_ragged_advance(kvr):  # noqa: F811
    cache = kvr.PagedKVCache(1, 3, 1, 64, num_pages=300, page_size=16, track_weights=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    for more in (700, [3, 0, 1]):
        cache.advance(more)
        T = 700 if more == 700 else 3
        k, v = (torch.randn(3, 1, T, 64, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
        cache.append(0, k, v)
    q = torch.randn(3, 4, 3, 64, device="cuda", generator=g).to(torch.bfloat16)
    out = cache.attention(0, q)
    for b, m in enumerate((3, 0, 1)):
        one = slice(b, b + 1)
        assert (out[b, :, :3 - m] == 0).all()
        total = cache.token_weights[0][b].double().sum().item()
        assert abs(total - 4 * m) <= 2 ** -14 * 4 * m            # the weights of m queries of 4 heads
        if m:
            want, size, _, _ = reference(q[one, :, 3 - m:], cache.key_pages[0], cache.value_pages[0],
                                         cache.block_table[one], cache.lengths[one])
            assert ((out[one, :, 3 - m:].double() - want).abs() <= (2 ** -8 + 2 ** -12) * size + 1e-7).all()


def test_refusals(kvr):  # noqa: F811
    q, k, v, table, n = make([50, 60], 12, 2, 128, 2, 16)
    nk = torch.zeros(2, 2, 2, 128, device="cuda", dtype=torch.bfloat16)
    for bad in (torch.zeros(2, device="cuda"), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32).cuda(),
                torch.zeros(2, 1, dtype=torch.int32).cuda(), torch.zeros(4, dtype=torch.int32).cuda()[::2]):
        with pytest.raises(ValueError):
            kvr.paged_decode_attention(q, k, v, table, n, new_counts=bad)
        with pytest.raises(ValueError):
            kvr.paged_append(nk, nk, k, v, table, n, new_counts=bad)
