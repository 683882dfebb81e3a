"""Paged attention where scores, values or lengths leave the ordinary range.
Tolerances as derived in test_gpu_paged.py."""
import pytest
import torch

from test_gpu_paged import check, kvr, make  # noqa: F401  (kvr: the fixture)

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
    from test_gpu_paged import reference

    q, k, v, table, n = data
    out, lse = kvr.paged_decode_attention(q, k, v, table, n, scale=1.0, return_lse=True)
    want, size, want_lse, _ = reference(q[few], k, v, table[few], n[few], scale=1.0)
    u = 2.0 ** -9 if q.dtype == torch.bfloat16 else 2.0 ** -12
    err = (out[few].double() - want).abs()
    assert (err <= (2 * u + 2 ** -12) * size + 1e-7).all(), f"out off by {(err / size).max().item():.2e}"
    assert (lse[few].double() - want_lse).abs().max().item() <= 2 ** -14
