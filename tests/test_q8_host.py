"""The 8-bit cache's C ABI and Python checks that need no GPU: struct layouts,
and descriptors that are refused before anything touches CUDA."""
import ctypes as ct

import pytest
import torch

from astc_kv_cuda import _lib as L


def _cache():
    c = L.AkvQ8Cache()
    c.format, c.block_tokens, c.batch, c.kv_heads, c.head_dim = L.AKV_Q8_INT8, 32, 2, 3, 64
    c.max_tokens = c.page_tokens = 128
    for s in (c.k, c.v):
        s.codes, s.scales = 4096, 4096
        s.stride_batch, s.stride_head, s.stride_token = 3 * 128 * 64, 128 * 64, 64
        s.scale_stride_batch, s.scale_stride_head = 12, 4
    return c


def _attention():
    d = L.AkvQ8AttnDesc()
    d.cache = _cache()
    d.q_heads, d.q_tokens, d.q_dtype, d.out_dtype = 9, 1, L.AKV_Q_BF16, L.AKV_Q_F32
    d.q_dev, d.out_dev = 4096, 4096
    d.q_stride[:] = (576, 576, 64)
    return d


def _evict():
    d = L.AkvQ8EvictDesc()
    d.src, d.dst = _cache(), _cache()
    for s in (d.dst.k, d.dst.v):
        s.codes, s.scales = 8192, 8192
    d.weights_dev, d.weights_stride, d.keep = 4096, 128, 64
    d.kept_dev, d.out_lens_dev, d.out_weights_dev, d.out_weights_stride = 4096, 4096, 4096, 64
    return d


def test_struct_sizes():
    lib = L.lib()
    for i, s in enumerate((L.AkvQ8Cache, L.AkvQ8StoreDesc, L.AkvQ8RestoreDesc, L.AkvQ8AttnDesc, L.AkvQ8EvictDesc)):
        assert lib.akv_q8_struct_size(i) == ct.sizeof(s)
    assert lib.akv_q8_struct_size(5) == 0


BAD_CACHES = [
    ("format", 2, 1), ("block_tokens", 48, 1), ("block_tokens", 8, 2), ("block_tokens", 0, 1), ("head_dim", 72, 2),
    ("head_dim", 272, 2), ("head_dim", 0, 1), ("kv_heads", 0, 1), ("max_tokens", 0, 1), ("page_tokens", 100, 1), ("batch", -1, 1),
]


@pytest.mark.parametrize("field,value,status", BAD_CACHES)
def test_every_call_refuses_a_bad_cache(field, value, status):
    lib = L.lib()
    a, e = _attention(), _evict()
    s, r = L.AkvQ8StoreDesc(), L.AkvQ8RestoreDesc()
    s.cache, r.cache = _cache(), _cache()
    s.tokens = r.tokens = 1
    for c in (a.cache, e.src, s.cache, r.cache):
        setattr(c, field, value)
    assert lib.akv_q8_attention_workspace(ct.byref(a)) == 0
    for fn, d in ((lib.akv_q8_attention, a), (lib.akv_q8_evict, e), (lib.akv_q8_store, s), (lib.akv_q8_restore, r)):
        assert fn(ct.byref(d), None) == status


def test_planes_are_checked():
    lib = L.lib()
    for side in ("k", "v"):
        for field, value in (("codes", None), ("codes", 4104), ("scales", None), ("scales", 4097), ("stride_head", 72),
                             ("stride_token", 65), ("stride_batch", 8), ("stride_page", 24)):
            d = _attention()
            setattr(getattr(d.cache, side), field, value)
            assert lib.akv_q8_attention(ct.byref(d), None) == 1, (side, field)
    d = _attention()
    d.cache.block_table_dev, d.cache.pages_per_seq, d.cache.num_pages = 4096, 1, 0
    assert lib.akv_q8_attention(ct.byref(d), None) == 1
    d.cache.num_pages, d.cache.max_tokens = 4, 129  # more tokens than the table has pages for
    assert lib.akv_q8_attention(ct.byref(d), None) == 1


def test_attention_refusals():
    lib = L.lib()
    assert lib.akv_q8_attention(None, None) == 1
    d = _attention()
    size = lib.akv_q8_attention_workspace(ct.byref(d))
    assert size >= 16
    assert lib.akv_q8_attention(ct.byref(d), None) == 6  # no workspace
    d.workspace_dev, d.workspace_bytes = 4096, size - 1
    assert lib.akv_q8_attention(ct.byref(d), None) == 6
    d.workspace_dev, d.workspace_bytes = 4100, size
    assert lib.akv_q8_attention(ct.byref(d), None) == 1
    for field, value in (("q_heads", 10), ("q_heads", 0), ("q_tokens", -1), ("q_dtype", 3), ("out_dtype", -1), ("split_tokens", 24),
                         ("split_tokens", -16), ("scale", float("nan")), ("scale", -1.0), ("scale", float("inf")), ("q_dev", None),
                         ("out_dev", None), ("q_dev", 4097), ("out_dev", 4100)):
        d = _attention()
        d.workspace_dev, d.workspace_bytes = 4096, 1 << 30
        setattr(d, field, value)
        assert lib.akv_q8_attention(ct.byref(d), None) == 1, (field, value)
    d = _attention()
    d.workspace_dev, d.workspace_bytes = 4096, 1 << 30
    d.weights_dev, d.weights_stride = 4096, 127
    assert lib.akv_q8_attention(ct.byref(d), None) == 1


def test_nothing_to_do_is_not_an_error():
    lib = L.lib()
    d = _attention()
    d.q_tokens = 0
    assert lib.akv_q8_attention(ct.byref(d), None) == 0
    s, r = L.AkvQ8StoreDesc(), L.AkvQ8RestoreDesc()
    s.cache, r.cache = _cache(), _cache()
    assert lib.akv_q8_store(ct.byref(s), None) == 0
    assert lib.akv_q8_restore(ct.byref(r), None) == 0


def test_store_and_restore_refusals():
    lib = L.lib()
    assert lib.akv_q8_store(None, None) == 1 and lib.akv_q8_restore(None, None) == 1
    for field, value in (("tokens", -1), ("dtype", 3), ("k_dev", None), ("v_dev", None), ("start_dev", None), ("k_dev", 4097)):
        s = L.AkvQ8StoreDesc()
        s.cache, s.tokens, s.dtype = _cache(), 4, L.AKV_Q_F16
        s.k_dev = s.v_dev = s.start_dev = 4096
        setattr(s, field, value)
        assert lib.akv_q8_store(ct.byref(s), None) == 1, field
    for field, value in (("tokens", -1), ("dtype", 3), ("k_dev", None), ("v_dev", 4104)):
        r = L.AkvQ8RestoreDesc()
        r.cache, r.tokens = _cache(), 4
        r.k_dev = r.v_dev = 4096
        setattr(r, field, value)
        assert lib.akv_q8_restore(ct.byref(r), None) == 1, field


def test_evict_refusals():
    lib = L.lib()
    assert lib.akv_q8_evict(None, None) == 1
    for field, value in (("keep", 0), ("keep", 129), ("sinks", -1), ("recent", -1), ("sinks", 65), ("weights_dev", None),
                         ("kept_dev", None), ("out_lens_dev", None), ("out_weights_dev", None), ("weights_stride", 127),
                         ("out_weights_stride", 63)):
        d = _evict()
        setattr(d, field, value)
        assert lib.akv_q8_evict(ct.byref(d), None) == 1, field
    for field, value in (("format", 1), ("batch", 1), ("kv_heads", 1), ("head_dim", 32)):
        d = _evict()
        setattr(d.dst, field, value)
        assert lib.akv_q8_evict(ct.byref(d), None) == 1, field
    d = _evict()
    d.dst.v.codes = d.src.v.codes
    assert lib.akv_q8_evict(ct.byref(d), None) == 1


def test_python_refuses_cpu_tensors_and_other_dtypes():
    from astc_kv_cuda import Q8Cache
    codes, scales = torch.zeros(1, 1, 64, 64, dtype=torch.int8), torch.zeros(1, 1, 1)
    with pytest.raises(ValueError):
        Q8Cache(codes, codes, scales, scales)
    with pytest.raises(ValueError):
        Q8Cache(codes.float(), codes.float(), scales, scales)
    with pytest.raises(ValueError):
        Q8Cache.zeros(1, 1, 64, 64, fmt="int4", device="cpu")


def test_evict_refuses_counts_of_weights_that_do_not_fit():
    lib = L.lib()
    for tokens in (-1, 63, 97):
        d = _evict()
        d.out_weights_stride, d.out_weights_tokens = 96, tokens
        assert lib.akv_q8_evict(ct.byref(d), None) == 1, tokens


def test_evict_within_a_pool_needs_two_tables():
    lib = L.lib()
    d = _evict()
    for side in ("k", "v"):
        getattr(d.dst, side).codes = getattr(d.src, side).codes
        getattr(d.dst, side).scales = getattr(d.src, side).scales
    for c in (d.src, d.dst):
        c.block_table_dev, c.pages_per_seq, c.num_pages, c.batch = 4096, 1, 8, 0  # a batch of none: nothing is launched
    assert lib.akv_q8_evict(ct.byref(d), None) == 1
    d.dst.block_table_dev = 8192
    assert lib.akv_q8_evict(ct.byref(d), None) == 0
    d.dst.block_table_dev, d.dst.max_tokens = None, 128
    assert lib.akv_q8_evict(ct.byref(d), None) == 1


def test_a_batch_of_none_needs_no_memory():
    """Empty tensors have no address; there is nothing to do, and that is not an error."""
    lib = L.lib()
    s, r, a, e = L.AkvQ8StoreDesc(), L.AkvQ8RestoreDesc(), _attention(), _evict()
    s.cache, r.cache = _cache(), _cache()
    s.tokens = r.tokens = 4
    for c in (s.cache, r.cache, a.cache, e.src, e.dst):
        c.batch = 0
        for side in (c.k, c.v):
            side.codes = side.scales = None
    a.q_dev = a.out_dev = e.weights_dev = e.kept_dev = e.out_lens_dev = e.out_weights_dev = None
    assert lib.akv_q8_attention_workspace(ct.byref(a)) >= 16
    for fn, d in ((lib.akv_q8_attention, a), (lib.akv_q8_evict, e), (lib.akv_q8_store, s), (lib.akv_q8_restore, r)):
        assert fn(ct.byref(d), None) == 0


@pytest.mark.parametrize("q_tokens,more", [(128, True), (512, False)])
def test_ragged_lengths_ask_for_more_splits_of_few_rows_only(q_tokens, more):
    """Partials take workspace. With rows for every SM, lengths do not change the splits."""
    lib = L.lib()
    d = _attention()
    d.cache.batch, d.cache.kv_heads, d.cache.head_dim, d.cache.max_tokens, d.cache.page_tokens = 4, 8, 128, 8192, 8192
    d.q_heads, d.q_tokens, d.out_dtype = 32, q_tokens, L.AKV_Q_BF16
    without = lib.akv_q8_attention_workspace(ct.byref(d))
    d.seq_lens_dev = 4096
    assert (lib.akv_q8_attention_workspace(ct.byref(d)) > without) == more


@pytest.mark.parametrize("head_dim,rows", [(64, 33), (128, 33), (144, 17), (256, 17)])
def test_rows_from_which_the_kernel_for_many_rows_is_taken(head_dim, rows):
    """It shows in the workspace: one step of that kernel has no partials, or two a row where two tiles share the rows."""
    lib = L.lib()
    for n in (rows - 1, rows):
        d = _attention()
        d.cache.batch, d.cache.kv_heads, d.cache.head_dim, d.cache.max_tokens = 1, 1, head_dim, 128
        d.q_heads, d.q_tokens, d.out_dtype = 1, n, L.AKV_Q_BF16
        parts = 2 * n if head_dim <= 128 else 0
        want = (parts * 8 + 15) // 16 * 16 + parts * head_dim * 4 + 16
        assert (lib.akv_q8_attention_workspace(ct.byref(d)) == want) == (n == rows)


def test_addresses_of_words_are_checked():
    """int32 and fp32 arrays on odd addresses would fault on the GPU."""
    lib = L.lib()

    def store():
        s = L.AkvQ8StoreDesc()
        s.cache, s.tokens, s.dtype = _cache(), 4, L.AKV_Q_F16
        s.k_dev = s.v_dev = s.start_dev = s.counts_dev = 4096
        return s

    def restore():
        r = L.AkvQ8RestoreDesc()
        r.cache, r.tokens = _cache(), 4
        r.k_dev = r.v_dev = r.start_dev = 4096
        return r

    def attention():
        d = _attention()
        d.workspace_dev, d.workspace_bytes = 4096, 1 << 30
        d.weights_stride = 128
        return d
    for make, fn, fields in ((store, lib.akv_q8_store, ("start_dev", "counts_dev")), (restore, lib.akv_q8_restore, ("start_dev",)),
                             (attention, lib.akv_q8_attention, ("seq_lens_dev", "q_lens_dev", "lse_dev", "weights_dev")),
                             (_evict, lib.akv_q8_evict, ("weights_dev", "kept_dev", "out_lens_dev", "out_weights_dev", "seq_lens_dev"))):
        for field in fields:
            d = make()
            setattr(d, field, 4098)
            assert fn(ct.byref(d), None) == 1, field
        for field in ("block_table_dev", "status_dev"):
            d = make()
            c = d.src if hasattr(d, "src") else d.cache
            c.pages_per_seq, c.num_pages = 1, 2
            setattr(c, field, 4098)
            assert fn(ct.byref(d), None) == 1, field
