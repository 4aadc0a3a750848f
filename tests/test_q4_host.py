"""The 4-bit cache's and the rotation's C ABI checks that need no GPU: struct
layouts, and descriptors that are refused before anything touches CUDA."""
import ctypes as ct

import pytest
import torch

from astc_kv_cuda import _lib as L


def _cache():
    c = L.AkvQ4Cache()
    c.batch, c.kv_heads, c.head_dim = 2, 3, 64
    c.max_tokens = c.page_tokens = 128
    for s in (c.k, c.v):
        s.codes, s.scales = 4096, 4096
        s.stride_batch, s.stride_head, s.stride_token = 3 * 128 * 32, 128 * 32, 32
        s.scale_stride_batch, s.scale_stride_head, s.scale_stride_group = 3 * 256, 256, 128
    return c


def _rotary():
    r = L.AkvRotary()
    r.table_dev, r.positions, r.rotary_dim, r.axes = 4096, 100, 64, 1
    return r


def _attention():
    d = L.AkvQ4AttnDesc()
    d.cache = _cache()
    d.q_heads, d.q_tokens, d.q_dtype, d.out_dtype = 9, 1, L.AKV_Q_BF16, L.AKV_Q_F32
    d.q_dev, d.out_dev = 4096, 4096
    d.q_stride[:] = (576, 576, 64)
    return d


def _append():
    d = L.AkvQ4AppendDesc()
    d.cache, d.rotary = _cache(), _rotary()
    d.tokens, d.dtype, d.q_heads = 4, L.AKV_Q_BF16, 9
    d.k_dev = d.v_dev = d.q_dev = d.q_out_dev = d.start_dev = 4096
    return d


def _rotate():
    d = L.AkvRotateDesc()
    d.rotary = _rotary()
    d.batch, d.tokens, d.heads, d.head_dim, d.dtype = 2, 4, 3, 64, L.AKV_Q_F16
    d.x_dev, d.out_dev, d.positions_dev = 4096, 8192, 4096
    return d


def test_struct_sizes():
    lib = L.lib()
    for i, s in enumerate((L.AkvQ4Cache, L.AkvQ4AppendDesc, L.AkvQ4RestoreDesc, L.AkvQ4AttnDesc)):
        assert lib.akv_q4_struct_size(i) == ct.sizeof(s)
    for i, s in enumerate((L.AkvRotary, L.AkvRotateDesc)):
        assert lib.akv_rotary_struct_size(i) == ct.sizeof(s)
    assert lib.akv_q4_struct_size(4) == lib.akv_rotary_struct_size(2) == 0


def test_no_descriptor():
    lib = L.lib()
    for fn in (lib.akv_q4_append, lib.akv_q4_restore, lib.akv_q4_attention, lib.akv_rotate):
        assert fn(None, None) == 1
    assert lib.akv_q4_attention_workspace(None) == 0


@pytest.mark.parametrize("field,value,status", [
    ("head_dim", 72, 2), ("head_dim", 48, 2), ("head_dim", 288, 2), ("head_dim", 0, 1), ("kv_heads", 0, 1), ("max_tokens", 0, 1),
    ("max_tokens", (1 << 30) + 1, 2), ("page_tokens", 100, 1), ("page_tokens", 8, 1), ("page_tokens", 0, 1), ("batch", -1, 1), ("batch", 40000, 2),
])
def test_every_call_refuses_a_bad_cache(field, value, status):
    lib = L.lib()
    a, s, r = _attention(), _append(), L.AkvQ4RestoreDesc()
    s.rotary = L.AkvRotary()
    s.q_dev = None
    r.cache = _cache()
    r.tokens = 1
    for c in (a.cache, s.cache, r.cache):
        setattr(c, field, value)
    assert lib.akv_q4_attention_workspace(ct.byref(a)) == 0
    for fn, d in ((lib.akv_q4_attention, a), (lib.akv_q4_append, s), (lib.akv_q4_restore, r)):
        assert fn(ct.byref(d), None) == status


def test_planes_are_checked():
    lib = L.lib()
    for side in ("k", "v"):
        for field, value in (("codes", None), ("codes", 4104), ("scales", None), ("scales", 4100), ("stride_head", 72), ("stride_token", 40),
                             ("stride_batch", 8), ("stride_page", 24), ("scale_stride_group", 130), ("scale_stride_head", 2),
                             ("scale_stride_batch", 1), ("scale_stride_page", 6)):
            d = _attention()
            setattr(getattr(d.cache, side), field, value)
            assert lib.akv_q4_attention(ct.byref(d), None) == 1, (side, field)
    d = _attention()
    d.cache.block_table_dev, d.cache.pages_per_seq, d.cache.num_pages = 4096, 1, 0
    assert lib.akv_q4_attention(ct.byref(d), None) == 1
    d.cache.num_pages, d.cache.max_tokens = 4, 129  # more tokens than the table has pages for
    assert lib.akv_q4_attention(ct.byref(d), None) == 1
    d = _attention()
    d.cache.status_dev = 4098
    assert lib.akv_q4_attention(ct.byref(d), None) == 1


@pytest.mark.parametrize("field,value,status", [
    ("q_heads", 0, 1), ("q_heads", 10, 1), ("q_tokens", -1, 1), ("q_dtype", 3, 1), ("out_dtype", -1, 1), ("split_tokens", 24, 1),
    ("split_tokens", -16, 1), ("scale", -1.0, 1), ("scale", float("nan"), 1), ("scale", float("inf"), 1), ("q_dev", None, 1), ("q_dev", 4097, 1),
    ("out_dev", None, 1), ("out_dev", 4104, 1), ("seq_lens_dev", 4098, 1), ("q_lens_dev", 4097, 1), ("lse_dev", 4098, 1), ("q_tokens", 1 << 22, 2),
    ("workspace_dev", None, 6),
])
def test_attention_refuses(field, value, status):
    d = _attention()
    setattr(d, field, value)
    assert L.lib().akv_q4_attention(ct.byref(d), None) == status


def test_attention_workspace():
    lib = L.lib()
    d = _attention()
    need = lib.akv_q4_attention_workspace(ct.byref(d))
    assert need >= 16
    d.workspace_dev, d.workspace_bytes = 4096, need - 1
    assert lib.akv_q4_attention(ct.byref(d), None) == 6
    d.workspace_dev, d.workspace_bytes = 4104, need
    assert lib.akv_q4_attention(ct.byref(d), None) == 1


@pytest.mark.parametrize("field,value", [
    ("tokens", -1), ("dtype", 3), ("k_dev", None), ("v_dev", None), ("start_dev", None), ("k_dev", 4097), ("v_dev", 4097), ("q_dev", 4097),
    ("start_dev", 4098), ("counts_dev", 4097), ("positions_dev", 4098), ("q_out_dev", None), ("q_out_dev", 4104), ("q_heads", 0),
])
def test_append_refuses(field, value):
    d = _append()
    setattr(d, field, value)
    assert L.lib().akv_q4_append(ct.byref(d), None) == 1


def test_append_without_a_table_takes_no_queries_or_positions():
    d = _append()
    d.rotary = L.AkvRotary()
    assert L.lib().akv_q4_append(ct.byref(d), None) == 1
    d.q_dev, d.positions_dev = None, 4096
    assert L.lib().akv_q4_append(ct.byref(d), None) == 1


@pytest.mark.parametrize("field,value,status", [
    ("table_dev", 4104, 1), ("positions", 0, 1), ("rotary_dim", 0, 1), ("rotary_dim", 63, 1), ("rotary_dim", 66, 1), ("rotary_dim", -2, 1),
    ("axes", 0, 1), ("axes", 9, 2),
])
def test_bad_tables(field, value, status):
    lib = L.lib()
    a, r = _append(), _rotate()
    for d in (a, r):
        setattr(d.rotary, field, value)
    assert lib.akv_q4_append(ct.byref(a), None) == status
    assert lib.akv_rotate(ct.byref(r), None) == status


def test_an_axis_outside_the_axes():
    lib = L.lib()
    a, r = _append(), _rotate()
    for d in (a, r):
        d.rotary.axis[31] = 1
    assert lib.akv_q4_append(ct.byref(a), None) == lib.akv_rotate(ct.byref(r), None) == 1


@pytest.mark.parametrize("field,value,status", [
    ("batch", -1, 1), ("tokens", -1, 1), ("heads", 0, 1), ("head_dim", 0, 1), ("head_dim", 32, 1), ("head_dim", 258, 2), ("dtype", 4, 1),
    ("x_dev", None, 1), ("out_dev", None, 1), ("positions_dev", None, 1), ("x_dev", 4097, 1), ("out_dev", 4097, 1), ("positions_dev", 4098, 1),
    ("status_dev", 4098, 1),
])
def test_rotate_refuses(field, value, status):
    d = _rotate()
    setattr(d, field, value)
    assert L.lib().akv_rotate(ct.byref(d), None) == status


def test_empty_calls_need_no_memory():
    lib = L.lib()
    a, s, r, t = _attention(), _append(), L.AkvQ4RestoreDesc(), _rotate()
    r.cache = _cache()
    r.tokens = 1
    for c in (a.cache, s.cache, r.cache):
        c.batch = 0
        c.k.codes = c.k.scales = c.v.codes = c.v.scales = None
    t.batch = 0
    s.k_dev = s.v_dev = s.q_dev = s.q_out_dev = s.start_dev = a.q_dev = a.out_dev = t.x_dev = t.out_dev = t.positions_dev = None
    for fn, d in ((lib.akv_q4_attention, a), (lib.akv_q4_append, s), (lib.akv_q4_restore, r), (lib.akv_rotate, t)):
        assert fn(ct.byref(d), None) == 0
    a, s, t = _attention(), _append(), _rotate()
    a.q_tokens = s.tokens = t.tokens = 0
    for fn, d in ((lib.akv_q4_attention, a), (lib.akv_q4_append, s), (lib.akv_rotate, t)):
        assert fn(ct.byref(d), None) == 0


def test_python_checks_that_need_no_gpu():
    from astc_kv_cuda import Q4Cache, Rotary
    codes = torch.zeros(1, 1, 16, 16, dtype=torch.uint8)
    scales = torch.zeros(1, 1, 1, 16, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        Q4Cache(codes, codes, scales, scales)
    with pytest.raises(ValueError, match="uint8"):
        Q4Cache(codes.to(torch.int8), codes, scales, scales)
    with pytest.raises(ValueError, match="CUDA"):
        Rotary(torch.zeros(4, 8, 2))
    for bad in (torch.zeros(4, 8), torch.zeros(4, 8, 3), torch.zeros(4, 8, 2, dtype=torch.float64), torch.zeros(4, 8, 4)[..., ::2]):
        with pytest.raises(ValueError, match="table"):
            Rotary(bad)
    for kw in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=258), dict(rotary_dim=8, sections=(1, 2)),
               dict(rotary_dim=8, sections=(4,), axes=[0] * 4), dict(rotary_dim=8, frequencies=torch.ones(3)), dict(rotary_dim=8, positions=0)):
        with pytest.raises(ValueError):
            Rotary.make(**{"positions": 4, "device": "cpu", **kw})
