"""What is written must not share memory with itself."""
import pytest
import torch

from test_gpu_paged import kvr, make  # noqa: F401  (kvr: the fixture)

pytestmark = pytest.mark.gpu


def test_expanded_tensors_are_refused_where_they_are_written(kvr):  # noqa: F811
    q, k, v, table, n = make([50, 60], 8, 2, 64, 1, 16)
    cap = table.shape[1] * 16
    one = torch.zeros(1, cap, device="cuda")
    flat = torch.zeros(2 * cap, device="cuda")
    for w in (one.expand(2, -1), flat.as_strided((2, cap), (cap - 1, 1)), flat[:1].expand(2, cap)):
        with pytest.raises(ValueError):
            kvr.paged_decode_attention(q, k, v, table, n, token_weights=w)
    for w in (one.repeat(2, 1), flat.view(2, cap), torch.zeros(2, cap + 3, device="cuda")[:, :cap]):
        kvr.paged_decode_attention(q, k, v, table, n, token_weights=w)
    kvr.paged_decode_attention(q[:1], k, v, table[:1], n[:1], token_weights=one.expand(1, -1))
    new = torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16, device="cuda")
    fresh = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
    for bad in (k[:1].expand(k.shape), k[:, :1].expand(k.shape), k[:, :, :1].expand(k.shape)):
        for pools in ((bad, v), (v, bad)):
            with pytest.raises(ValueError):
                kvr.paged_append(new, new, *pools, table, n)
            with pytest.raises(ValueError):
                kvr.paged_evict(*pools, table, n, flat.view(2, cap), fresh, keep=16)
    # reading them is no matter
    want = kvr.paged_decode_attention(q, k[:, :1].repeat(1, 2, 1, 1), v, table, n)
    assert torch.equal(kvr.paged_decode_attention(q, k[:, :1].expand(k.shape), v, table, n), want)
