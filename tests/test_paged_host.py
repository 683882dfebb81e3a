"""The paged cache's page accounting and the new operators' fake shapes and
refusals, without a GPU."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import kv_reduce_b200.ops  # noqa: F401  (registers torch.ops.kvr.*)
from kv_reduce_b200.paged import PagedKVCache


def held(cache):
    """Every page is either free or one sequence's, and the tables say so."""
    pages = [p for seq in cache._pages for p in seq]
    assert sorted(pages + cache._free) == list(range(cache.num_pages))
    for b, seq in enumerate(cache._pages):
        assert cache.block_table[b].tolist() == seq + [-1] * (cache.max_pages - len(seq))
        assert len(seq) == -(-cache._lengths[b] // cache.page_size)
    assert cache.lengths.tolist() == cache.seq_lengths()


def test_pages_follow_the_lengths():
    c = PagedKVCache(2, 3, 2, 64, num_pages=20, page_size=8, max_pages=9, device="cpu")
    held(c)
    for step in (5, [3, 0, 11], 8, [0, 1, 0]):
        c.advance(step)
        held(c)
    assert c.seq_lengths() == [16, 14, 24] and c.get_seq_length() == 24 and c.free_pages() == 20 - 7
    c.crop([16, 9, 1])
    held(c)
    c.crop(8)
    held(c)
    assert c.seq_lengths() == [8, 8, 1]
    with pytest.raises(ValueError):
        c.crop([9, 8, 1])
    with pytest.raises(ValueError):
        c.crop([0, 0])
    with pytest.raises(ValueError):
        c.advance(-1)
    with pytest.raises(ValueError):
        c.advance([1, 1])
    with pytest.raises(ValueError):
        c.advance([66, 0, 0])                # max_pages
    with pytest.raises(ValueError):
        c.advance(56)                        # 24 pages wanted, 20 there
    held(c)
    assert c.seq_lengths() == [8, 8, 1]      # a refused step changes nothing
    c.crop(0)
    held(c)
    assert c.free_pages() == 20


def test_eviction_checks():
    c = PagedKVCache(1, 1, 1, 64, num_pages=4, page_size=4, device="cpu")
    with pytest.raises(ValueError):
        c.evict(2)                           # no weights
    c = PagedKVCache(1, 1, 1, 64, num_pages=4, page_size=4, device="cpu", track_weights=True)
    c.advance(12)
    for kw in (dict(keep=0), dict(keep=4, recent=3, first=2), dict(keep=4, recent=-1)):
        with pytest.raises(ValueError):
            c.evict(**kw)
    assert c.evict(12) is False
    with pytest.raises(ValueError):
        c.evict(8)                           # two fresh pages wanted, one there
    held(c)
    with pytest.raises(ValueError):
        PagedKVCache(1, 0, 1, 64, num_pages=4)


def test_fake_shapes():
    with FakeTensorMode():
        q = torch.empty(2, 12, 3, 128, dtype=torch.bfloat16, device="cuda")
        pages = torch.empty(9, 2, 16, 128, dtype=torch.bfloat16, device="cuda")
        table = torch.empty(2, 4, dtype=torch.int32, device="cuda")
        lengths = torch.empty(2, dtype=torch.int32, device="cuda")
        w = torch.empty(2, 64, device="cuda")
        assert torch.ops.kvr.paged_append(q[:, :2], q[:, :2], pages, pages, table, lengths) is None
        out, lse = torch.ops.kvr.paged_attention(q, pages, pages, table, lengths, return_lse=True)
        assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (2, 12, 3) and lse.dtype == torch.float32
        kept, n, kw = torch.ops.kvr.paged_evict(pages, pages, table, lengths, w, table, 20, 4, 1)
        assert kept.shape == kw.shape == (2, 20) and kept.dtype == n.dtype == torch.int32 and n.shape == (2,)
        t = torch.empty(2, 5, 100, dtype=torch.bfloat16, device="cuda")
        x = torch.empty(2, 4, dtype=torch.int64, device="cuda")
        tokens, acc, prob = torch.ops.kvr.verify_draft(t, None, x, None, None, 0.0)
        assert tokens.shape == (2, 5) and tokens.dtype == torch.int64 and acc.dtype == torch.int32
        assert prob.shape == (2, 4) and prob.dtype == torch.float32


def test_no_cpu_fallback():
    import kv_reduce_b200 as kvr

    q, pages = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 8, 64, dtype=torch.bfloat16)
    table, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (lambda: kvr.paged_decode_attention(q, pages, pages, table, n),
                 lambda: kvr.paged_append(q, q, pages, pages, table, n),
                 lambda: kvr.paged_evict(pages, pages, table, n, torch.zeros(1, 8), table, keep=4),
                 lambda: kvr.verify_draft_tokens(torch.zeros(1, 2, 8), None, torch.zeros(1, 1, dtype=torch.long),
                                                 temperature=0)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_c_abi_refusals(built_lib):
    """Bad arguments are rejected before any CUDA call."""
    from kv_reduce_b200 import _lib

    lib = _lib.load()
    a = _lib.PagedAttentionArgs()
    a.batch, a.q_heads, a.kv_heads, a.head_dim, a.new_tokens, a.page_size = 1, 12, 2, 128, 1, 16
    a.table_width, a.num_pages, a.num_sms, a.scale = 4, 8, 148, 1.0
    assert lib.kvr_paged_attention_plan(a, None, None, None) == _lib.KVR_OK
    a.query = a.out = a.lengths = a.block_table = a.key_pages = a.value_pages = 256
    assert lib.kvr_paged_attention(a, None) == _lib.KVR_ERR_WORKSPACE
    a.q_b_stride = 4
    assert lib.kvr_paged_attention(a, None) == _lib.KVR_ERR_MISALIGNED
    a.q_b_stride, a.head_dim = 0, 96
    assert lib.kvr_paged_attention_plan(a, None, None, None) == _lib.KVR_ERR_UNSUPPORTED
    a.head_dim, a.q_heads = 128, 13
    assert lib.kvr_paged_attention_plan(a, None, None, None) == _lib.KVR_ERR_INVALID_ARGUMENT
    a.q_heads, a.table_width, a.page_size = 12, 1 << 20, 1 << 11
    assert lib.kvr_paged_attention_plan(a, None, None, None) == _lib.KVR_ERR_UNSUPPORTED
    e = _lib.PagedEvictArgs()
    e.batch, e.kv_heads, e.head_dim, e.page_size, e.keep = 1, 2, 64, 16, 8
    e.table_width, e.num_pages, e.new_table_width, e.first, e.recent = 4, 8, 1, 5, 4
    assert lib.kvr_paged_evict(e, None) == _lib.KVR_ERR_INVALID_ARGUMENT
    e.first = e.recent = 0
    assert lib.kvr_paged_evict(e, None) == _lib.KVR_ERR_INVALID_ARGUMENT      # null pointers
    e.keep = 40
    assert lib.kvr_paged_evict(e, None) == _lib.KVR_ERR_CAPACITY
    e.keep = 8                               # lengths in place (refused before a pointer is read)
    e.lengths = e.new_lengths = e.kept = e.new_weights = e.block_table = e.new_block_table = 64
    e.token_weights = e.key_pages = e.value_pages = 128
    assert lib.kvr_paged_evict(e, None) == _lib.KVR_ERR_INVALID_ARGUMENT
    v = _lib.VerifyArgs()
    v.batch, v.draft_tokens, v.vocab, v.temperature = 1, 2, 100, -1.0
    assert lib.kvr_verify(v, None) == _lib.KVR_ERR_INVALID_ARGUMENT
    v.temperature = 1.0
    assert lib.kvr_verify(v, None) == _lib.KVR_ERR_INVALID_ARGUMENT           # null pointers
    v.dtype = 3
    assert lib.kvr_verify(v, None) == _lib.KVR_ERR_UNSUPPORTED
