"""Verification of drafted tokens against the rule in 64 bits.

accept_prob is a ratio of two softmaxes in fp32: the exponents' products
carry at most 2^-24 * 60 each and the sums 2^-22, 2^-16 in all (relative).
A decision that 64 bits leave within that of the other side (u against a, or
the race's best two) may fall either way: such sequences are not compared."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
EDGE = 2.0 ** -16


@pytest.fixture(scope="module")
def kvr(built_lib):
    import kv_reduce_b200

    return kv_reduce_b200


def make(B, K, V, dtype, temp=1.0, seed=0, spread=0.7, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randn(B, K + 1, V + pad, device="cuda", generator=g) * 2
    d = t[:, :K] + spread * torch.randn(B, K, V + pad, device="cuda", generator=g)
    t, d = t.to(dtype)[..., :V], d.to(dtype)[..., :V]
    x = torch.distributions.utils.probs_to_logits(torch.softmax(d.double() / max(temp, 1e-3), -1)) if K else d.double()
    e = torch.empty(B, K, V, device="cuda").exponential_(generator=g)
    tokens = (x - e.double().log()).argmax(-1)
    u = torch.rand(B, K, device="cuda", generator=g)
    noise = torch.empty(B, V, device="cuda").exponential_(generator=g).clamp_min(1e-30)
    return t, d, tokens, u, noise


def rule(t, d, tokens, u, noise, temp, n_draft=None):
    """(tokens, accepted, accept_prob, sure) in 64 bits; `sure`: no decision is near an edge."""
    B, K1, V = t.shape
    K = K1 - 1
    out, acc = torch.full((B, K1), -1, dtype=torch.long), torch.zeros(B, dtype=torch.int32)
    prob, sure = torch.zeros(B, K, dtype=torch.float64), torch.ones(B, dtype=torch.bool)
    for b in range(B):
        n = K if n_draft is None else min(max(int(n_draft[b]), 0), K)
        at = n
        for k in range(n):
            x = int(tokens[b, k])
            if temp == 0:
                row = t[b, k].double()
                prob[b, k] = float(x == int((row == row.max()).nonzero()[0, 0]))
                no = prob[b, k] == 0
            else:
                lp, lq = (torch.log_softmax(z[b, k].double() / temp, -1) for z in (t, d))
                a = 0.0
                if 0 <= x < V and lp[x] > -math.inf:
                    a = min(1.0, math.exp(min(0.0, float(lp[x] - lq[x]))))
                prob[b, k] = a
                sure[b] &= abs(float(u[b, k]) - a) > EDGE or a == 1.0
                no = not float(u[b, k]) < a
            if no:
                at = k
                break
        acc[b] = at
        out[b, :at] = tokens[b, :at].cpu()
        if temp == 0:
            row = t[b, at].double()
            out[b, at] = int((row == row.max()).nonzero()[0, 0])
            continue
        p = torch.softmax(t[b, at].double() / temp, -1)
        w = p
        if at < n:
            w = (p - torch.softmax(d[b, at].double() / temp, -1)).clamp_min(0)
            if w.max() < EDGE * 1e-3:
                sure[b] = False
        score = (w / noise[b].double()).nan_to_num(0.0)
        if score.max() > 0:
            out[b, at] = int((score == score.max()).nonzero()[0, 0])
            top = score.topk(min(2, V)).values
            sure[b] &= len(top) < 2 or bool(top[1] < top[0] * (1 - EDGE)) or bool(top[1] == top[0])
    return out, acc, prob, sure


def check(kvr, data, temp, n_draft=None, least=0.9):
    t, d, tokens, u, noise = data
    r = kvr.verify_draft_tokens(t, d, tokens, u, noise, temperature=temp, draft_lengths=n_draft)
    out, acc, prob, sure = rule(t, d, tokens, u, noise, temp, n_draft)
    assert r.tokens.dtype == torch.int64 and r.accepted.dtype == torch.int32 and r.accept_prob.dtype == torch.float32
    assert sure.double().mean() >= least
    assert torch.equal(r.tokens.cpu()[sure], out[sure])
    assert torch.equal(r.accepted.cpu()[sure], acc[sure])
    err = (r.accept_prob.cpu().double() - prob).abs()[sure]
    assert (err <= EDGE * prob[sure] + 1e-30).all()
    again = kvr.verify_draft_tokens(t, d, tokens, u, noise, temperature=temp, draft_lengths=n_draft)
    for a, b in zip(r, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [2, 7, 64, 1000, 4099, 32001])
@pytest.mark.parametrize("temp", [0.0, 0.7, 1.0])
def test_sizes_and_types(kvr, dtype, V, temp):
    check(kvr, make(9, 4, V, dtype, temp, seed=V), temp)


@pytest.mark.parametrize("B,K", [(1, 1), (1, 8), (3, 0), (70, 3), (400, 1), (2, 17)])
@pytest.mark.parametrize("temp", [0.0, 1.0])
def test_batches_and_drafts(kvr, B, K, temp):
    check(kvr, make(B, K, 513, torch.bfloat16, temp, seed=B + K), temp)


@pytest.mark.parametrize("V", [70000, 151001])
def test_large_vocabulary(kvr, V):
    check(kvr, make(4, 3, V, torch.bfloat16, 0.8, seed=V), 0.8)
    check(kvr, make(2, 3, V, torch.float32, 0.0, seed=V), 0.0)


@pytest.mark.parametrize("pad", [1, 3, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_padded_rows(kvr, pad, dtype):
    """Logits cut from wider rows: any row stride, any alignment."""
    for temp in (0.0, 1.0):
        check(kvr, make(5, 3, 1001, dtype, temp, seed=pad, pad=pad), temp)
    t, d, tokens, u, noise = make(5, 3, 999, dtype, 1.0, seed=pad)
    swapped = t.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(5, 3, 1998, dtype=dtype, device="cuda")
    wide[..., ::2] = d
    a = kvr.verify_draft_tokens(t, d, tokens, u, noise)
    b = kvr.verify_draft_tokens(swapped, wide[..., ::2], tokens.int(), u.t().contiguous().t(), noise)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


@pytest.mark.parametrize("temp", [0.0, 1.0])
def test_ragged_drafts(kvr, temp):
    n = torch.tensor([0, 1, 2, 3, 4, 5, -1, 99], dtype=torch.int32, device="cuda")
    check(kvr, make(8, 5, 300, torch.bfloat16, temp, seed=1, spread=0.05), temp, n)


def test_filtered_logits(kvr):
    """-inf outside the target's and the draft's top tokens."""
    t, d, tokens, u, noise = make(40, 4, 2000, torch.float32, 1.0, seed=3)
    t = torch.where(t < t.topk(5).values[..., -1:], -math.inf, t)
    d = torch.where(d < d.topk(20).values[..., -1:], -math.inf, d)
    tokens = (d.double() - torch.empty_like(d).exponential_().double().log()).argmax(-1)
    check(kvr, (t, d, tokens, u, noise), 1.0)
    low = torch.finfo(torch.float32).min                     # masks of the lowest value
    check(kvr, (t.clamp_min(low), d.clamp_min(low), tokens, u, noise), 1.0)


def test_acceptance_of_equal_and_disjoint_models(kvr):
    t, d, tokens, u, noise = make(30, 4, 700, torch.bfloat16, 1.0, seed=5)
    r = kvr.verify_draft_tokens(t, t[:, :4].contiguous(), tokens, u, noise)
    assert (r.accepted == 4).all() and torch.equal(r.tokens[:, :4], tokens) and (r.accept_prob == 1).all()
    t, d = t.clone(), d.clone()
    t[..., :350], d[..., 350:] = -math.inf, -math.inf
    tokens %= 350
    r = kvr.verify_draft_tokens(t, d, tokens, u, noise)
    assert (r.accepted == 0).all() and (r.tokens[:, 0] >= 350).all() and (r.accept_prob == 0).all()


def test_rows_without_weight_and_bad_tokens(kvr):
    t, d, tokens, u, noise = make(6, 2, 100, torch.bfloat16, 1.0, seed=6)
    t[0] = -math.inf
    tokens[1, 0], tokens[2, 0] = -5, 100
    for temp in (1.0, 0.0):
        r = kvr.verify_draft_tokens(t, d, tokens, u, noise, temperature=temp)
        assert (r.accepted[1:3] == 0).all() and (r.tokens[1:3, 0] >= 0).all()
        if temp:
            assert r.accepted[0] == 0 and r.tokens[0].tolist() == [-1, -1, -1]
    check(kvr, (t[3:], d[3:], tokens[3:], u[3:], noise[3:]), 1.0, least=0.5)
    nothing_left = kvr.verify_draft_tokens(t[3:], t[3:, :2].contiguous(), tokens[3:], torch.ones_like(u[3:]), noise[3:])
    assert (nothing_left.accepted == 0).all() and (nothing_left.tokens[:, 0] >= 0).all()   # drawn from p


def test_ties_go_to_the_lowest_index(kvr):
    V = 5000
    t = torch.zeros(3, 2, V, dtype=torch.bfloat16, device="cuda")
    t[1, :, 1234:] = 1
    t[2] = -math.inf
    tokens = torch.tensor([[0], [1234], [0]], device="cuda")
    r = kvr.verify_draft_tokens(t, None, tokens, temperature=0)
    assert r.tokens.tolist() == [[0, 0], [1234, 1234], [0, 0]] and r.accepted.tolist() == [1, 1, 1]
    ones = torch.ones(3, V, device="cuda")
    r = kvr.verify_draft_tokens(t[:2], t[:2, :1].contiguous(), tokens[:2], torch.zeros(2, 1, device="cuda"), ones[:2])
    assert r.tokens.tolist() == [[0, 0], [1234, 1234]]


def test_tokens_follow_the_target(kvr):
    """The first token of many rounds has the target's distribution, whatever the draft."""
    B, V = 40000, 8
    g = torch.Generator(device="cuda").manual_seed(7)
    row_t, row_d = (torch.randn(V, device="cuda", generator=g) for _ in range(2))
    t, d = row_t.expand(B, 2, V).contiguous(), row_d.expand(B, 1, V).contiguous()
    tokens = torch.multinomial(torch.softmax(row_d, -1), B, replacement=True, generator=g)[:, None]
    u = torch.rand(B, 1, device="cuda", generator=g)
    noise = torch.empty(B, V, device="cuda").exponential_(generator=g)
    r = kvr.verify_draft_tokens(t, d, tokens, u, noise)
    p = torch.softmax(row_t.double(), -1).cpu()
    share = torch.bincount(r.tokens[:, 0].cpu(), minlength=V).double() / B
    assert ((share - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all()
    assert (r.accepted == 1).any() and (r.accepted == 0).any()


def test_stream_and_graph(kvr):
    t, d, tokens, u, noise = make(6, 3, 3001, torch.bfloat16, 1.0, seed=8)
    want = kvr.verify_draft_tokens(t, d, tokens, u, noise)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = kvr.verify_draft_tokens(t, d, tokens, u, noise)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        in_graph = kvr.verify_draft_tokens(t, d, tokens, u, noise)
    for _ in range(3):
        graph.replay()
    for a, b, c in zip(want, got, in_graph):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_refusals(kvr):
    t, d, x, u, e = make(3, 2, 50, torch.bfloat16)
    f = kvr.verify_draft_tokens
    for args in [(t.cpu(), d, x, u, e), (t[0], d, x, u, e), (t.double(), d, x, u, e), (t, d.float(), x, u, e),
                 (t, d[:, :1], x, u, e), (t, d[..., :49], x, u, e), (t, None, x, u, e), (t, d, x[:, :1], u, e),
                 (t, d, x.float(), u, e), (t, d, x.cpu(), u, e), (t, d, x, None, e), (t, d, x, u[:2], e),
                 (t, d, x, u.double(), e), (t, d, x, u, None), (t, d, x, u, e[:, :49]), (t, d, x, u, e.cpu()),
                 (t[..., :0], d[..., :0], x, u, e[:, :0])]:
        with pytest.raises(ValueError):
            f(*args)
    for temp in (-1.0, math.inf, math.nan, 1e-60, 1e-38):
        with pytest.raises(ValueError):
            f(t, d, x, u, e, temperature=temp)
    with pytest.raises(ValueError):
        f(t, d, x, u, e, draft_lengths=torch.zeros(3, device="cuda"))
    r = f(t[:0], d[:0], x[:0], u[:0], e[:0])
    assert r.tokens.shape == (0, 3) and r.accepted.shape == (0,) and r.accept_prob.shape == (0, 2)
