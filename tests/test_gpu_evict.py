"""Eviction by accumulated weight against a sort on the host; everything it
returns is copied or counted, so all of it has to be equal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kvr(built_lib):
    import kv_reduce_b200

    return kv_reduce_b200


def make(lengths, H, D, page, keep, seed=0, weights="random", dtype=torch.bfloat16, layout="heads"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B = len(lengths)
    need = [-(-n // page) for n in lengths]
    fresh = -(-keep // page)
    total = sum(need) + B * fresh + 2
    shape = (total, page, H, D) if layout == "tokens" else (total, H, page, D)
    k, v = (torch.randn(shape, device="cuda", generator=g).to(dtype) for _ in range(2))
    if layout == "tokens":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    order = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    table = torch.full((B, max(need + [1])), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    new_table = order[at:at + B * fresh].view(B, fresh).contiguous()
    cap = table.shape[1] * page
    w = torch.rand(B, cap + 5, device="cuda", generator=g)
    if weights == "ties":
        w = (w * 4).floor()
    elif weights == "equal":
        w = torch.full_like(w, 0.5)
    elif weights == "wide":
        w = torch.exp((w - 0.5) * 160)            # down to denormals, up to 1e34
        w[:, ::7] = 0
        w[:, 3::11] = -0.0
        w[:, 5::13] = -w[:, 5::13]
    elif weights == "odd":
        w[:, ::5], w[:, 1::50], w[:, 2::5] = -math.inf, math.inf, torch.finfo(torch.float32).min
        w[:, 4::97] = math.nan
    return k, v, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), w, new_table


def check(kvr, data, keep, recent, first):
    k, v, table, lengths, w, new_table = data
    page = k.shape[2]
    wk, wv = k.clone(), v.clone()
    B, host = len(lengths), w.cpu()
    want = torch.full((B, keep), -1, dtype=torch.int32)
    want_w = torch.zeros(B, keep)
    for b, n in enumerate(lengths.tolist()):
        kept = list(range(n))
        if n > keep:
            forced = [j for j in range(n) if j < first or j >= n - recent]
            x = host[b].tolist()
            rest = sorted((j for j in range(first, n - recent)),
                          key=lambda j: (0 if math.isnan(x[j]) else 1, 0 if math.isnan(x[j]) else -x[j], j))
            kept = sorted(forced + rest[:keep - first - recent])
        want[b, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
        want_w[b, :len(kept)] = host[b][kept]
        if kept:
            src, dst = torch.tensor(kept, device="cuda"), torch.arange(len(kept), device="cuda")
            for pool in (wk, wv):
                pool[new_table[b].long()[dst // page], :, dst % page] = pool[table[b].long()[src // page], :, src % page]
    kept, new_lengths, new_w = kvr.paged_evict(k, v, table, lengths, w, new_table, keep=keep, recent=recent, first=first)
    assert torch.equal(new_lengths.cpu(), lengths.cpu().clamp_max(keep))
    assert torch.equal(kept.cpu(), want)
    assert torch.equal(new_w.cpu().view(torch.int32), want_w.view(torch.int32))
    assert torch.equal(k, wk) and torch.equal(v, wv)


@pytest.mark.parametrize("weights", ["random", "ties", "equal", "wide", "odd"])
@pytest.mark.parametrize("keep,recent,first", [(64, 0, 0), (64, 64, 0), (64, 60, 4), (64, 10, 3), (1, 0, 0), (500, 100, 7)])
def test_selection(kvr, weights, keep, recent, first):
    lengths = [0, 1, 63, 64, 65, 100, 777, 1500]
    check(kvr, make(lengths, 2, 64, 16, keep, seed=keep, weights=weights), keep, recent, first)


@pytest.mark.parametrize("lengths", [[5000], [40000, 39999, 1], [3000] * 40, [9000, 100] * 40, [90000]])
@pytest.mark.parametrize("weights", ["random", "ties"])
def test_long_and_many(kvr, lengths, weights):
    """One CTA to a cluster of eight per sequence; slices that end anywhere."""
    check(kvr, make(lengths, 1, 64, 32, 1024, seed=len(lengths), weights=weights), 1024, 200, 4)


@pytest.mark.parametrize("page", [1, 7, 16, 24, 100])
@pytest.mark.parametrize("H,D,layout", [(8, 64, "heads"), (2, 128, "tokens"), (3, 8, "heads"), (1, 256, "heads")])
def test_layouts(kvr, page, H, D, layout):
    check(kvr, make([300, 41, 120], H, D, page, 100, seed=page, dtype=torch.float16, layout=layout), 100, 30, 2)


def test_no_copy_of_bad_pages(kvr):
    k, v, table, lengths, w, new_table = make([300, 300], 2, 64, 16, 64, seed=3)
    bad_new, bad_old = new_table.clone(), table.clone()
    bad_new[0] = k.shape[0]
    bad_old[1] = -1
    wk, wv = k.clone(), v.clone()
    kept, _, _ = kvr.paged_evict(k, v, bad_old, lengths, w, bad_new, keep=64)
    assert torch.equal(k, wk) and torch.equal(v, wv) and (kept >= 0).all()


def test_capture_and_attention_after(kvr):
    """In a CUDA graph; attention over the new pages sees the kept tokens."""
    data = make([300, 500], 2, 64, 16, 128, seed=3)
    k, v, table, lengths, w, new_table = data
    kvr.paged_evict(k, v, table, lengths, w, new_table, keep=128, recent=16)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept, new_lengths, _ = kvr.paged_evict(k, v, table, lengths, w, new_table, keep=128, recent=16)
    w.mul_(-1)
    g.replay()
    q = torch.randn(2, 4, 1, 64, device="cuda").to(torch.bfloat16)
    out = kvr.paged_decode_attention(q, k, v, new_table, new_lengths)
    for b in range(2):
        j = kept[b].long()
        kk, vv = (p[table[b].long()[j // 16], :, j % 16].double() for p in (k, v))
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", q[b, :, 0].double().view(2, 2, 64), kk) / 8, -1)
        want = torch.einsum("hgn,nhd->hgd", p, vv).reshape(4, 64)
        assert (out[b, :, 0].double() - want).abs().max() < 2 ** -8 * vv.abs().max()


def test_refusals(kvr):
    k, v, table, lengths, w, new_table = make([300, 300], 2, 64, 16, 64)
    ok = dict(keep=64, recent=4, first=1)
    for args, kw in [((k.cpu(), v, table, lengths, w, new_table), ok), ((k, v, table, lengths, w.cpu(), new_table), ok),
                     ((k, v, table, lengths, w.double(), new_table), ok), ((k, v, table, lengths, w[:, :100], new_table), ok),
                     ((k, v, table, lengths, w[:1], new_table), ok), ((k, v, table, lengths, w, new_table.long()), ok),
                     ((k, v, table, lengths, w, new_table[:, :3]), ok), ((k, v, table, lengths, w, new_table[:1]), ok),
                     ((k, v, table, lengths, w, new_table), dict(keep=0)),
                     ((k, v, table, lengths, w, new_table), dict(keep=64, recent=60, first=5)),
                     ((k, v, table, lengths, w, new_table), dict(keep=64, recent=-1)),
                     ((k, v[:, :, :4], table, lengths, w, new_table), ok)]:
        with pytest.raises(ValueError):
            kvr.paged_evict(*args, **kw)
    big = torch.zeros(1, 20001, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        kvr.paged_evict(k, v, big, lengths[:1], torch.zeros(1, 320016, device="cuda"), new_table[:1], **ok)
