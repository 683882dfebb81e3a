"""Paged attention where scores, values or lengths leave the ordinary range.
Tolerances as derived in test_gpu_paged.py."""
import math

import pytest
import torch

from test_gpu_paged import check, kvr, make, reference  # noqa: F401  (kvr: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("gap", [12.0, 17.0, 18.0, 22.0])
@pytest.mark.parametrize("HQ,H,D,T", [(4, 1, 64, 1), (12, 2, 128, 1), (12, 2, 128, 5), (8, 1, 128, 9)])
def test_one_token_outweighs_the_others(kvr, HQ, H, D, T, gap, dtype):  # noqa: F811
    """An attention sink: the first token `gap` above the others' scores, its
    value 0, so that the output is what the others' small weights carry.  Long
    sequences in one CTA's range, and one that many CTAs share."""
    for lengths in ([4095] * (400 // H), [20000]):
        q, k, v, table, n = make(lengths, HQ, H, D, T, 64, dtype, seed=int(gap), garbage=False)
        first = table[:, 0].long()
        q.zero_()
        q[..., 0] = 8
        k.zero_()
        k[first, :, 0, 0] = gap / 8
        for value in ("ones", "random"):
            if value == "ones":
                keep = v.clone()
                v.fill_(1)
            else:
                v.copy_(keep)
            v[first, :, 0] = 0
            few = slice(0, 3)          # the formula on a few sequences, which all compute the same thing
            check(kvr, (q, k, v, table, n), scale=1.0) if len(lengths) == 1 else \
                check_few(kvr, (q, k, v, table, n), few)


def check_few(kvr, data, few):  # noqa: F811
    """The whole batch runs; `few` sequences are compared with the formula."""
    q, k, v, table, n = data
    out, lse = kvr.paged_decode_attention(q, k, v, table, n, scale=1.0, return_lse=True)
    want, size, want_lse, _ = reference(q[few], k, v, table[few], n[few], scale=1.0)
    u = 2.0 ** -9 if q.dtype == torch.bfloat16 else 2.0 ** -12
    err = (out[few].double() - want).abs()
    assert (err <= (2 * u + 2 ** -12) * size + 1e-7).all(), f"out off by {(err / size).max().item():.2e}"
    assert (lse[few].double() - want_lse).abs().max().item() <= 2 ** -14


def far_scores(lengths, HQ, H, D, T, dtype, size, seed, page=16, width=None):
    """Scores of about `size` (either sign), products of two numbers that the
    type holds, so exact: a few equal ones on top and the others a step or
    more below."""
    q, k, v, table, n = make(lengths, HQ, H, D, T, page, dtype, seed=seed, garbage=False, max_pages=width)
    root = 2.0 ** round(math.log2(abs(size)) / 2)
    q.zero_()
    k.zero_()
    q[..., 3] = root
    step = torch.randint(0, 4, k.shape[:3], device="cuda", generator=torch.Generator("cuda").manual_seed(seed))
    step = torch.where(torch.rand(step.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) < 0.9,
                       step + 1, 0)
    k[..., 3] = (root * (1.5 - step / 64) if size > 0 else -root * (1 + step / 64)).to(k.dtype)
    return q, k, v, table, n


@pytest.mark.parametrize("dtype,size", [("bf16", 2.0 ** x) for x in (20, 30, 60, 118)] +
                         [("bf16", -2.0 ** x) for x in (20, 30, 60, 118)] + [("fp16", 2.0 ** 28), ("fp16", -2.0 ** 28)])
@pytest.mark.parametrize("HQ,H,D,T,window", [(12, 2, 128, 1, 0), (8, 2, 64, 3, 0), (12, 2, 128, 3, 200)])
def test_scores_far_from_zero(kvr, HQ, H, D, T, window, dtype, size):  # noqa: F811
    """Only differences of scores count, however large the scores: down to
    those below -1e30, and where fp32's spacing is more than the exponents'
    range."""
    lengths = [1500, 130, 129, 1, 0, 9000]
    q, k, v, table, n = far_scores(lengths, HQ, H, D, T, dtype, size, seed=HQ)
    out, lse = kvr.paged_decode_attention(q, k, v, table, n, scale=1.0, window=window, return_lse=True)
    want, _, want_lse, _ = reference(q, k, v, table, n, window, scale=1.0)
    u = 2.0 ** -9 if dtype == "bf16" else 2.0 ** -12
    _, size_v, _, _ = reference(q, k, v.abs(), table, n, window, scale=1.0)
    assert ((out.double() - want).abs() <= (2 * u + 2 ** -12) * size_v + 1e-7).all()
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert ((lse.double() - want_lse).abs() <= 2.0 ** -22 * want_lse.abs() + 2 ** -14)[~empty].all()


@pytest.mark.parametrize("dtype,size", [("bf16", 2.0 ** 20), ("bf16", -2.0 ** 30), ("bf16", 2.0 ** 118), ("fp16", 2.0 ** 28)])
@pytest.mark.parametrize("page", [16, 2])
@pytest.mark.parametrize("HQ,H,D,T", [(12, 2, 128, 5), (16, 2, 128, 9), (16, 2, 64, 9)])
def test_scores_far_from_zero_in_wide_tables(kvr, HQ, H, D, T, page, dtype, size):  # noqa: F811
    """The same in tiles of 32 and 64 rows, and with rows copied one by one."""
    q, k, v, table, n = far_scores([1500, 130, 1, 4000], HQ, H, D, T, dtype, size, HQ, page, 160000 // page)
    w = torch.zeros(4, table.shape[1] * page, device="cuda")
    out, lse = kvr.paged_decode_attention(q, k, v, table, n, scale=1.0, return_lse=True, token_weights=w)
    want, _, want_lse, want_w = reference(q, k, v, table, n, scale=1.0)
    size_v = reference(q, k, v.abs(), table, n, scale=1.0)[1]
    u = 2.0 ** -9 if dtype == "bf16" else 2.0 ** -12
    assert ((out.double() - want).abs() <= (2 * u + 2 ** -12) * size_v + 1e-7).all()
    empty = want_lse == -math.inf
    assert ((lse.double() - want_lse).abs() <= 2.0 ** -22 * want_lse.abs() + 2 ** -14)[~empty].all()
    assert ((w.double() - want_w).abs() <= 2 ** -14 * want_w + 1e-6).all()


@pytest.mark.parametrize("dtype,size", [("bf16", x) for x in (2.0 ** 12, 2.0 ** 20, -2.0 ** 30, 2.0 ** 118, -2.0 ** 118)] +
                         [("fp16", 2.0 ** 14), ("fp16", -2.0 ** 28)])
@pytest.mark.parametrize("HQ,H,D,T", [(12, 2, 128, 1), (8, 2, 64, 3)])
def test_weights_of_scores_far_from_zero(kvr, HQ, H, D, T, dtype, size):  # noqa: F811
    """Each token's share, not rounded to the spacing of the scores."""
    q, k, v, table, n = far_scores([1500, 130, 129, 1, 0, 9000], HQ, H, D, T, dtype, size, seed=HQ)
    w = torch.full((6, table.shape[1] * 16), 0.25, device="cuda")
    kvr.paged_decode_attention(q, k, v, table, n, scale=1.0, token_weights=w)
    want = reference(q, k, v, table, n, scale=1.0)[3]
    assert ((w.double() - 0.25 - want).abs() <= 2 ** -14 * want + 1e-6).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("HQ,H,D,T", [(12, 2, 128, 1), (8, 2, 64, 4), (12, 2, 128, 5), (8, 1, 128, 9)])
def test_infinite_values_that_are_seen(kvr, HQ, H, D, T, dtype):  # noqa: F811
    """They reach the output as what they are: an infinity of its sign, NaN
    where both signs meet or a value is NaN; other elements are untouched."""
    lengths = [300, 129, 40, 9000]
    q, k, v, table, n = make(lengths, HQ, H, D, T, 16, dtype, seed=T)
    clean = kvr.paged_decode_attention(q, k, v, table, n)
    bad = [(0, math.inf), (1, -math.inf), (2, math.nan), (3, math.inf), (3, -math.inf)]
    for b, length in enumerate(lengths):
        for at in (5, length // 2, length - T):           # tokens that every query sees
            for c, x in bad[:4]:
                v[table[b, at // 16].long(), :, at % 16, 10 * c] = x
        v[table[b, 3 // 16].long(), :, 3, 30] = -math.inf
    out = kvr.paged_decode_attention(q, k, v, table, n)
    assert (out[..., 0] == math.inf).all() and (out[..., 10] == -math.inf).all()
    assert out[..., 20].isnan().all() and out[..., 30].isnan().all()
    others = [i for i in range(D) if i not in (0, 10, 20, 30)]
    assert torch.equal(out[..., others], clean[..., others])


@pytest.mark.parametrize("HQ,H,D,T", [(12, 2, 128, 1), (12, 2, 128, 9), (8, 1, 64, 33)])
def test_sequences_longer_than_a_short_table(kvr, HQ, H, D, T):  # noqa: F811
    """NaN for every query of such a sequence, also where the table holds fewer
    tokens than there are queries, or none."""
    q, k, v, table, n = make([20, 30, 8], HQ, H, D, T, 4, seed=T)
    for width in (0, 1, 2):
        for window in (0, 5):
            out, lse = kvr.paged_decode_attention(q, k, v, table[:, :width], n, window=window, return_lse=True)
            assert out[:2].isnan().all() and lse[:2].isnan().all()
            if width == 2:                               # the last one fits, whoever its neighbours are
                alone = kvr.paged_decode_attention(q[2:], k, v, table[2:, :2], n[2:], window=window)
                u = 2.0 ** -7
                assert torch.allclose(out[2:].float(), alone.float(), rtol=u, atol=u) and not alone.isnan().any()
            else:
                assert out[2].isnan().all()


@pytest.mark.parametrize("HQ,H,D,T", [(12, 2, 128, 200), (8, 2, 64, 131), (4, 4, 128, 300), (7, 1, 64, 150)])
def test_chunks_of_a_prompt(kvr, HQ, H, D, T):  # noqa: F811
    """Hundreds of new tokens, as the target's hook sends them."""
    check(kvr, make([1000, T, T - 40, 1, 0], HQ, H, D, T, 16, seed=T))
    check(kvr, make([777, T + 3], HQ, H, D, T, 24, "fp16", seed=T), 90, 5)
