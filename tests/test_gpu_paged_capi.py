"""The paged operators through the C ABI, where torch's checks do not stand in front."""
import pytest
import torch

from test_gpu_paged import kvr, make  # noqa: F401  (kvr: the fixture)

pytestmark = pytest.mark.gpu


def attention(q, k, v, table, n, window=0, sinks=0, weights=False):
    from kv_reduce_b200 import _lib
    from ctypes import byref, c_size_t

    lib, a = _lib.load(), _lib.PagedAttentionArgs()
    out, w = torch.empty_like(q, memory_format=torch.contiguous_format), None
    a.query, a.q_b_stride, a.q_h_stride, a.q_t_stride = q.data_ptr(), *q.stride()[:3]
    a.key_pages, a.key_page_stride, a.key_head_stride, a.key_row_stride = k.data_ptr(), *k.stride()[:3]
    a.value_pages, a.value_page_stride, a.value_head_stride, a.value_row_stride = v.data_ptr(), *v.stride()[:3]
    a.block_table, a.table_stride, a.table_width, a.num_pages = table.data_ptr(), table.stride(0), table.shape[1], k.shape[0]
    a.lengths, a.out = n.data_ptr(), out.data_ptr()
    a.batch, a.q_heads, a.new_tokens, a.head_dim = q.shape
    a.kv_heads, a.page_size, a.window, a.sinks, a.scale = k.shape[1], k.shape[2], window, sinks, q.shape[3] ** -0.5
    if weights:
        w = torch.zeros(q.shape[0], table.shape[1] * k.shape[2], device="cuda")
        a.token_weights, a.weights_b_stride = w.data_ptr(), w.stride(0)
    sizes = [c_size_t() for _ in range(3)]
    assert lib.kvr_paged_attention_plan(a, *map(byref, sizes)) == _lib.KVR_OK
    ws, cnt, sc = sizes[0].value, sizes[1].value, sizes[2].value
    buffers = [torch.empty(ws, dtype=torch.uint8, device="cuda"), torch.zeros(cnt, dtype=torch.int32, device="cuda"),
               torch.empty(max(sc, 16), dtype=torch.uint8, device="cuda")]
    a.workspace, a.workspace_bytes, a.counters, a.scores, a.scores_bytes = (
        buffers[0].data_ptr(), ws, buffers[1].data_ptr(), buffers[2].data_ptr(), sc)
    assert lib.kvr_paged_attention(a, torch.cuda.current_stream().cuda_stream) == _lib.KVR_OK
    torch.cuda.synchronize()
    assert not buffers[1].any()
    return out, w


@pytest.mark.parametrize("window,sinks", [((1 << 31) - 1, 0), ((1 << 31) - 1, (1 << 31) - 1), (200, (1 << 31) - 1),
                                          ((1 << 30) + 1, 5)])
def test_windows_and_sinks_near_2_to_the_31(kvr, window, sinks):  # noqa: F811
    """A window or sinks that cover every token: no mask at all."""
    for HQ, H, D, T in ((12, 2, 128, 1), (8, 2, 64, 4)):
        data = make([1500, 3, 400], HQ, H, D, T, 16, seed=T)
        want, want_w = attention(*data, weights=True)
        got, got_w = attention(*data, window, sinks, weights=True)
        assert torch.equal(got, want)
        n = data[4]
        for b in range(3):
            assert torch.equal(got_w[b, :n[b]], want_w[b, :n[b]])
