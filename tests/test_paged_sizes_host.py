"""Sizes near 2^31 at the C entries, refused before any CUDA call."""


def test_evict_keep(built_lib):
    from kv_reduce_b200 import _lib

    lib = _lib.load()
    e = _lib.PagedEvictArgs()
    e.batch, e.kv_heads, e.head_dim, e.page_size = 1, 2, 64, 16
    e.table_width, e.num_pages, e.new_table_width = 4, 8, 4
    for keep, status in ((1 << 30, _lib.KVR_ERR_INVALID_ARGUMENT),          # null pointers, a later check
                         ((1 << 30) + 1, _lib.KVR_ERR_UNSUPPORTED), ((1 << 31) - 1, _lib.KVR_ERR_UNSUPPORTED)):
        e.keep = keep
        assert lib.kvr_paged_evict(e, None) == status
