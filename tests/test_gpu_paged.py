"""Paged append and attention against the formulas in 64 bits.

Tolerances.  out: one rounding to the pages' type (at most 2u |o|, u = 2^-9
for bf16 and 2^-12 for fp16, and |o| <= sum p|v|); the scores carry an fp32
error of a few 2^-24 * sum |q k| * scale, which 2^-12 covers for the |q.k|
here (sum |q k| * scale < 300):  (2u + 2^-12) * sum p|v|.  lse and weights
are fp32: 2^-14 absolute on the log covers the same score error, and
relatively on each weight."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def kvr(built_lib):
    import kv_reduce_b200

    return kv_reduce_b200


def make(lengths, HQ, H, D, T, page, dtype="bf16", seed=0, layout="heads", extra=3, garbage=True, max_pages=None):
    """Pages, table and queries; every row that no token uses holds NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, B = DTYPES[dtype], len(lengths)
    need = [-(-n // page) for n in lengths]
    total = sum(need) + extra
    width = max_pages if max_pages is not None else max(need + [1]) + 1
    shape = (total, H, page, D)

    def pool():
        x = torch.randn(shape, device="cuda", generator=g).to(dt)
        if layout == "tokens":        # [num_pages, page, H, D] in memory
            return x.transpose(1, 2).contiguous().transpose(1, 2)
        return x

    if layout == "interleaved":       # keys and values of a page side by side
        both = torch.randn(total, 2, H, page, D, device="cuda", generator=g).to(dt)
        k, v = both[:, 0], both[:, 1]
    else:
        k, v = pool(), pool()
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    used = torch.zeros(total, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lengths):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        j = torch.arange(n, device="cuda")
        used[table[b].long()[j // page], j % page] = True
    if garbage:
        k.masked_fill_(~used[:, None, :, None], math.nan)
        v.masked_fill_(~used[:, None, :, None], math.nan)
    q = torch.randn(B, T, HQ, D, device="cuda", generator=g).to(dt).transpose(1, 2)
    return q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


def reference(q, k, v, table, lengths, window=0, sinks=0, scale=None):
    """Row by row in 64 bits: out, sum p|v|, lse, and each token's weight."""
    B, HQ, T, D = q.shape
    H, page = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, HQ, T, D, dtype=torch.float64, device="cuda")
    size, lse = torch.zeros_like(out), torch.full((B, HQ, T), -math.inf, dtype=torch.float64, device="cuda")
    weights = torch.zeros(B, table.shape[1] * page, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lengths.tolist()):
        for t in range(T):
            i = n - T + t
            j = torch.arange(max(i + 1, 0), device="cuda")
            if window:
                j = j[(j > i - window) | (j < sinks)]
            if not len(j):
                continue
            pages = table[b].long()[j // page]
            kk, vv = k[pages, :, j % page].double(), v[pages, :, j % page].double()      # [n, H, D]
            s = torch.einsum("hgd,nhd->hgn", q[b, :, t].double().view(H, HQ // H, D), kk) * scale
            lse[b, :, t] = torch.logsumexp(s, -1).reshape(HQ)
            p = torch.softmax(s, -1)
            out[b, :, t] = torch.einsum("hgn,nhd->hgd", p, vv).reshape(HQ, D)
            size[b, :, t] = torch.einsum("hgn,nhd->hgd", p, vv.abs()).reshape(HQ, D)
            weights[b, j] += p.sum((0, 1))
    return out, size, lse, weights


def check(kvr, data, window=0, sinks=0, scale=None):
    q, k, v, table, lengths = data
    want, size, want_lse, want_w = reference(q, k, v, table, lengths, window, sinks, scale)
    w = torch.full((q.shape[0], table.shape[1] * k.shape[2]), 0.25, device="cuda")
    out, lse = kvr.paged_decode_attention(q, k, v, table, lengths, window=window, sinks=sinks, scale=scale,
                                          token_weights=w, return_lse=True)
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    u = 2.0 ** -9 if q.dtype == torch.bfloat16 else 2.0 ** -12
    err = (out.double() - want).abs()
    assert not out.isnan().any()
    assert (err <= (2 * u + 2 ** -12) * size + 1e-7).all(), f"out off by {(err / (size + 1e-9)).max().item():.2e}"
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert (lse.double() - want_lse)[~empty].abs().max().item() <= 2 ** -14 if (~empty).any() else True
    assert ((w.double() - 0.25 - want_w).abs() <= 2 ** -14 * want_w + 1e-6).all()
    again = kvr.paged_decode_attention(q, k, v, table, lengths, window=window, sinks=sinks, scale=scale)
    assert torch.equal(again, out)          # the same bits, with the weights or without, on every call


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("HQ,H,D", [(12, 2, 128), (32, 8, 64), (8, 8, 128), (7, 1, 64), (40, 2, 128)])
@pytest.mark.parametrize("T", [1, 5])
def test_ragged_lengths(kvr, HQ, H, D, T, dtype):
    check(kvr, make([1, 17, 64, 65, 0, 300, 1029, 128, 5], HQ, H, D, T, 16, dtype, seed=T))


@pytest.mark.parametrize("page", [1, 2, 3, 4, 8, 12, 24, 64, 100, 256])
@pytest.mark.parametrize("layout", ["heads", "tokens", "interleaved"])
def test_page_sizes_and_layouts(kvr, page, layout):
    check(kvr, make([129, 700, 31], 12, 2, 128, 2, page, layout=layout, seed=page))
    check(kvr, make([129, 700, 31], 8, 4, 64, 1, page, layout=layout, seed=page + 1))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (64, 0), (100, 5), (128, 64), (257, 130), (511, 1), (5000, 3)])
@pytest.mark.parametrize("T", [1, 4])
def test_window_and_sinks(kvr, window, sinks, T):
    lengths = [1, 2, 63, 64, 65, 128, 400, 1000, 1537, 0]
    check(kvr, make(lengths, 12, 2, 128, T, 16, seed=window + T), window, sinks)
    check(kvr, make(lengths, 8, 2, 64, T, 24, "fp16", seed=window + T), window, sinks)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,HQ,H", [(1, 18, 1), (5, 12, 2), (4, 16, 2), (9, 16, 2), (33, 8, 1)])
def test_wide_tables_and_batches(kvr, T, HQ, H, D):
    """Enough room for tiles of more than 16 rows: by the table's width (few
    tokens in use), and by the batch."""
    check(kvr, make([3, 40, 333, 0, 129], HQ, H, D, T, 16, seed=T, max_pages=4000))
    check(kvr, make([3, 40, 333], HQ, H, D, T, 12, "fp16", seed=T, max_pages=8000), 40000, 3)
    lengths = [(i * 37) % 300 for i in range(1200 // H)]
    check(kvr, make(lengths, HQ, H, D, T, 16, seed=T + 1), 130, 5)


@pytest.mark.parametrize("page", [1, 2, 3, 10])
@pytest.mark.parametrize("T,HQ,H,D", [(5, 12, 2, 128), (9, 8, 1, 128), (33, 8, 1, 128), (9, 8, 1, 64)])
def test_small_pages_in_wide_tables(kvr, T, HQ, H, D, page):
    """Rows copied one by one into rings of every length."""
    check(kvr, make([3, 1040, 333, 0, 129], HQ, H, D, T, page, seed=T + page, max_pages=60000 // page))
    check(kvr, make([2000, 40], HQ, H, D, T, page, seed=page, max_pages=150000 // page), 70000, 3)


@pytest.mark.parametrize("T,HQ,H", [(8, 6, 1), (9, 16, 2), (11, 6, 1), (16, 8, 1), (33, 8, 1), (3, 64, 1)])
def test_many_rows(kvr, T, HQ, H):
    """48 to 264 query rows per KV head: every row-tile count; queries before
    the sequence's start where T is larger than it."""
    check(kvr, make([3, 40, 333], HQ, H, 128, T, 16, seed=T))
    check(kvr, make([3, 40, 333], HQ, H, 64, T, 16, seed=T), 70, 2)


@pytest.mark.parametrize("lengths", [[20000], [1], [0], [9000, 1, 1, 1], [4097] * 9, [50] * 700])
def test_splits_and_joins(kvr, lengths):
    """One long sequence cut over the whole GPU, one that no cut helps, and
    more sequences than CTAs."""
    check(kvr, make(lengths, 12, 2, 128, 1, 32, seed=len(lengths)))


def test_scale_and_large_scores(kvr):
    data = make([500, 77], 12, 2, 128, 1, 16, seed=5)
    check(kvr, data, scale=0.3)
    check(kvr, data, scale=-0.05)
    check(kvr, data, scale=0.0)


def test_empty_batch_and_capacity(kvr):
    q, k, v, table, lengths = make([5], 12, 2, 128, 1, 16)
    out = kvr.paged_decode_attention(q[:0], k, v, table[:0], lengths[:0])
    assert out.shape == (0, 12, 1, 128)
    # a table of no pages: every sequence is empty
    out, lse = kvr.paged_decode_attention(q, k, v, table[:, :0].contiguous(), lengths * 0, return_lse=True,
                                          token_weights=torch.zeros(1, 0, device="cuda"))
    assert out.abs().max().item() == 0 and (lse == -math.inf).all()


def test_bad_pages_and_lengths_give_nan(kvr):
    q, k, v, table, lengths = make([100, 100, 100, 100], 12, 2, 128, 1, 16, seed=2)
    good = kvr.paged_decode_attention(q, k, v, table, lengths)
    bad = table.clone()
    bad[1, 3], bad[2, 0] = -1, k.shape[0]
    out, lse = kvr.paged_decode_attention(q, k, v, bad, lengths, return_lse=True)
    assert torch.equal(out[[0, 3]], good[[0, 3]])
    assert out[[1, 2]].isnan().all() and lse[[1, 2]].isnan().all()
    # outside the window the page is not looked at
    out = kvr.paged_decode_attention(q, k, v, bad, lengths, window=20)
    assert not out.isnan().any()
    over = lengths.clone()
    over[3] = table.shape[1] * 16 + 1
    over[0] = -7
    out = kvr.paged_decode_attention(q, k, v, table, over)
    assert out[3].isnan().all() and out[0].abs().max().item() == 0 and torch.equal(out[1:3], good[1:3])


@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("bad", [math.inf, math.nan, -math.inf])
def test_nonfinite_values_where_masked(kvr, bad, window):
    """A drafted token's NaN or infinite key and value reach the queries that
    see it and no other."""
    T = 4
    for D, H in ((128, 2), (64, 2)):
        q, k, v, table, lengths = make([200, 131, 66], 12, H, D, T, 16, seed=9)
        ref = kvr.paged_decode_attention(q, k, v, table, lengths, window=window, sinks=1)
        for pool in (k, v):
            for b, n in enumerate([200, 131, 66]):
                j = n - 2                                  # seen by the last two queries
                pool[table[b, j // 16].long(), :, j % 16, 5] = bad
        out = kvr.paged_decode_attention(q, k, v, table, lengths, window=window, sinks=1)
        u = 2.0 ** -7
        assert torch.allclose(out[:, :, :2].float(), ref[:, :, :2].float(), rtol=u, atol=u)
        assert not out[:, :, :2].isnan().any()
        if window:                                         # the first token of the window's start
            q, k, v, table, lengths = make([200, 131, 90], 12, H, D, T, 16, seed=9)
            ref = kvr.paged_decode_attention(q, k, v, table, lengths, window=window)
            for b, n in enumerate([200, 131, 90]):
                j = n - T - window + 1                     # seen by the first query only
                v[table[b, j // 16].long(), :, j % 16, 5] = bad
            out = kvr.paged_decode_attention(q, k, v, table, lengths, window=window)
            assert torch.allclose(out[:, :, 1:].float(), ref[:, :, 1:].float(), rtol=u, atol=u)
            assert not out[:, :, 1:].isnan().any() and not out[:, :, 0, 5].isfinite().any()


def test_offsets_past_32_bits(kvr):
    """Pages behind the first 2^32 elements of a pool."""
    H, page, D = 2, 64, 128
    n_pages = (1 << 32) // (H * page * D) + 40
    pool = torch.empty(n_pages, H, page, D, dtype=torch.bfloat16, device="cuda")
    q, k, v, table, lengths = make([500, 900], 12, H, D, 1, page, seed=4)
    last = n_pages - k.shape[0]
    pool[last:] = k
    far = torch.where(table >= 0, table + last, table)
    want = kvr.paged_decode_attention(q, k, v, table, lengths)
    vpool = pool[last - 5:last - 5 + 1].expand(1, H, page, D)    # noqa: F841  (keeps the pool's tail in use)
    got = kvr.paged_decode_attention(q, pool, pool, far, lengths)
    same = kvr.paged_decode_attention(q, k, k, table, lengths)
    assert torch.equal(got, same) and want.shape == got.shape
    new = torch.randn(2, H, 1, D, device="cuda").to(torch.bfloat16)
    kvr.paged_append(new, new, pool, pool, far, lengths)
    assert torch.equal(pool[far[0, 499 // page].long(), :, 499 % page], new[0, :, 0])


@pytest.mark.parametrize("layout", ["heads", "tokens", "interleaved"])
@pytest.mark.parametrize("T", [1, 6])
def test_append(kvr, layout, T):
    q, k, v, table, lengths = make([3, 16, 17, 100, 0], 12, 2, 128, T, 16, layout=layout, seed=T, garbage=False)
    g = torch.Generator(device="cuda").manual_seed(1)
    nk = torch.randn(5, T, 2, 128, device="cuda", generator=g).to(torch.bfloat16).transpose(1, 2)
    nv = torch.randn(5, 2, T, 128, device="cuda", generator=g).to(torch.bfloat16)
    wk, wv = k.clone(), v.clone()
    for b, n in enumerate(lengths.tolist()):
        for t in range(T):
            j = n - T + t
            if j >= 0:
                wk[table[b, j // 16].long(), :, j % 16] = nk[b, :, t]
                wv[table[b, j // 16].long(), :, j % 16] = nv[b, :, t]
    kvr.paged_append(nk, nv, k, v, table, lengths)
    assert torch.equal(k, wk) and torch.equal(v, wv)
    # pages outside the pool and positions past the table are skipped
    bad = torch.full_like(table, k.shape[0])
    bad[0] = -1
    kvr.paged_append(nk, nv, k, v, bad, lengths)
    kvr.paged_append(nk, nv, k, v, table, lengths + 16 * table.shape[1] + T)
    assert torch.equal(k, wk) and torch.equal(v, wv)


def test_other_stream_and_graph(kvr):
    q, k, v, table, lengths = make([900, 333], 12, 2, 128, 1, 16, seed=8, garbage=False)
    nk = torch.randn(2, 2, 1, 128, device="cuda").to(torch.bfloat16)

    def step():
        kvr.paged_append(nk, nk, k, v, table, lengths)
        return kvr.paged_decode_attention(q, k, v, table, lengths)

    want = step().clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in (900, 512, 20):                    # the lengths are read on the device at each replay
        lengths.copy_(torch.tensor([n, n // 2], dtype=torch.int32))
        graph.replay()
        replayed = out.clone()
        # bit for bit; 450 tokens are more than the second sequence has pages for: NaN from both
        assert torch.equal(replayed.view(torch.int16), step().view(torch.int16))


def test_refusals(kvr):
    q, k, v, table, lengths = make([50, 60], 12, 2, 128, 1, 16)
    att = kvr.paged_decode_attention
    cases = [
        (q.cpu(), k, v, table, lengths), (q, k.cpu(), v, table, lengths), (q, k, v, table.cpu(), lengths),
        (q[0], k, v, table, lengths), (q.float(), k, v, table, lengths), (q, k, v.half(), table, lengths),
        (q, k, v[:, :, :8], table, lengths), (q, k[:, :1].expand(-1, 5, -1, -1), v[:, :1].expand(-1, 5, -1, -1), table, lengths),
        (q[..., :64], k, v, table, lengths), (q[..., :32], k[..., :32], v[..., :32], table, lengths),
        (q, k, v, table.long(), lengths), (q, k, v, table, lengths.long()), (q[:1], k, v, table, lengths),
        (q, k, v, table[:1], lengths), (q[:, :, :0], k, v, table, lengths),
        (q, k[..., ::2].repeat(1, 1, 1, 2)[..., 1:65], v[..., :64], table, lengths),
    ]
    for args in cases:
        with pytest.raises(ValueError):
            att(*args)
    for kw in (dict(window=-1), dict(window=4, sinks=-1), dict(token_weights=torch.zeros(2, 8, device="cuda")),
               dict(token_weights=torch.zeros(2, 1000, device="cuda", dtype=torch.float64))):
        with pytest.raises(ValueError):
            att(q, k, v, table, lengths, **kw)
    nk = torch.zeros(2, 2, 1, 128, device="cuda", dtype=torch.bfloat16)
    for bad in (nk.half(), nk[:1], nk[:, :1], nk[..., :64], nk.cpu()):
        with pytest.raises(ValueError):
            kvr.paged_append(bad, bad, k, v, table, lengths)
    assert not att(q, k, v, table, lengths).isnan().any()      # nothing of it left a mark
