"""Calls on the 8-bit cache that are prepared once and run again, on other
streams, and in memory that they share."""
import ctypes as ct

import pytest
import torch

from test_gpu_q8 import half_step, make, plain_choice, values_of, MOST

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("T,keep,room", [(300, 64, 128), (300, 64, 65), (9000, 500, 5000), (50, 64, 96)])
def test_evict_again_after_decoding(cuda, T, keep, room, graph):
    """The weights that decoding adds past the kept tokens are gone after the next eviction."""
    from astc_kv_cuda import Q8Attention, Q8Cache, Q8Evict
    cache, _, _ = make(2, 2, T, 64, seed=T)
    dst = Q8Cache.zeros(2, 2, room, 64, block_tokens=32)
    w = torch.rand(2, 2, cache.max_tokens, device="cuda")
    lens = torch.tensor([T, T // 3], dtype=torch.int32, device="cuda")
    call = Q8Evict(cache, dst, w, lens, keep=keep, sinks=2, recent=8)
    call.weights.fill_(float("nan"))
    call.run()
    torch.cuda.synchronize()
    again = call.run
    if graph:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call.run()
        again = g.replay
    for step in range(2):
        q = torch.randn(2, 8, 64, device="cuda").bfloat16()
        Q8Attention(q, dst, torch.full((2,), room, dtype=torch.int32, device="cuda"), weights=call.weights).run()
        assert (call.weights[:, :, min(keep, T // 3):] > 0).any()
        w.copy_(torch.rand_like(w))
        again()
        torch.cuda.synchronize()
        for b, n in enumerate(lens.tolist()):
            m = min(n, keep)
            assert int(call.lens[b]) == m and not call.weights[b, :, m:].any() and (call.kept[b, :, m:] == -1).all()
            for h in range(2):
                at = torch.as_tensor(plain_choice(w[b, h].cpu().numpy(), n, keep, 2, 8), device="cuda").long()
                assert torch.equal(call.weights[b, h, :m], w[b, h, at])


def test_evict_writes_the_weights_it_is_told_to(cuda):
    """Rows of out_weights that are further apart than they are long: what lies between them stays."""
    from astc_kv_cuda import Q8Cache, Q8Evict, _lib as L
    cache, _, _ = make(2, 2, 100, 32, seed=1)
    dst = Q8Cache.zeros(2, 2, 64, 32, block_tokens=32)
    w = torch.rand(2, 2, cache.max_tokens, device="cuda")
    call = Q8Evict(cache, dst, w, torch.tensor([100, 20], dtype=torch.int32, device="cuda"), keep=40)
    for tokens, end in ((0, 40), (40, 40), (57, 57), (80, 80)):
        out = torch.full((2, 2, 80), 7.0, device="cuda")
        call.desc.out_weights_dev, call.desc.out_weights_stride, call.desc.out_weights_tokens = out.data_ptr(), 80, tokens
        L.check(L.lib().akv_q8_evict(ct.byref(call.desc), None), "q8_evict")
        torch.cuda.synchronize()
        assert (out[0, :, :40] < 1).all() and not out[0, :, 40:end].any() and not out[1, :, 20:end].any()
        assert (out[:, :, end:] == 7).all()


def small_calls():
    """By name, what builds a call on a small cache, with an input that only the call holds: each call that owns memory."""
    from astc_kv_cuda import Q8Attention, Q8Cache, Q8Evict, Q8Restore
    cache, _, _ = make(2, 2, 4096, 64, seed=3)
    q0 = torch.randn(2, 8, 64, device="cuda").bfloat16()
    w0 = torch.rand(2, 2, 4096, device="cuda")

    def attention():
        q = q0.clone()
        return Q8Attention(q, cache)

    def restore():
        start = torch.full((2,), 7, dtype=torch.int32, device="cuda")
        return Q8Restore(cache, start, 64)

    def evict():
        w = w0.clone()
        return Q8Evict(cache, Q8Cache.zeros(2, 2, 1024, 64, block_tokens=32), w, keep=1024)
    return {"attention": attention, "restore": restore, "evict": evict}


def results(out):
    return list(out) if isinstance(out, tuple) else [out]


@pytest.mark.parametrize("op", ["attention", "restore", "evict"])
def test_other_stream_waits_for_the_memory(cuda, op):
    """Work that was given to the building stream before still writes to memory that the call got from its allocator."""
    build = small_calls()[op]
    want = [t.clone() for t in results(build().run())]
    side = torch.cuda.Stream()
    for _ in range(3):
        torch.cuda.synchronize()
        torch.cuda._sleep(100_000_000)
        junk = [torch.full_like(t, 77) for t in want for _ in range(3)]
        del junk
        got = results(build().run(side))
        side.synchronize()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("explicit", [False, True])
@pytest.mark.parametrize("op", ["attention", "restore", "evict"])
def test_memory_stays_until_the_other_stream_is_done(cuda, op, explicit):
    """The call and what it reads are dropped while the stream that it was given has not begun with it."""
    build = small_calls()[op]
    want = [t.clone() for t in results(build().run())]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        call = build()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)
            if not explicit:
                got = results(call.run())
        if explicit:
            got = results(call.run(side))
        sizes = [t.numel() * t.element_size() for t in call._tensors]
        del call
        junk = [torch.full((n,), 77, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(2)]
        torch.cuda.synchronize()
        del junk
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_first_run_inside_a_graph(cuda):
    """A call built outside runs for the first time while a graph is captured."""
    for op, build in small_calls().items():
        want = [t.clone() for t in results(build().run())]
        call = build()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = results(call.run())
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), op


def check_packed(src_values, dst, kept, lens):
    """`dst` holds the kept rows, each block under a scale of its own."""
    for b, n in enumerate(lens):
        for h in range(dst.kv_heads):
            at = kept[b, h, :n].long()
            for got, values in zip(values_of(dst), src_values):
                rows = values[b, h, at]
                pad = torch.zeros(-(-n // dst.block_tokens) * dst.block_tokens, dst.head_dim, dtype=torch.float64, device="cuda")
                pad[:n] = rows
                sc = (pad.view(-1, dst.block_tokens, dst.head_dim).abs().amax((1, 2)) / MOST[dst.fmt]).repeat_interleave(dst.block_tokens)[:n, None]
                assert ((got[b, h, :n] - rows).abs() <= half_step(rows, sc, dst.fmt) * (1 + 2.0 ** -10)).all()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_evict_into_other_pages_of_the_pool(cuda, fmt):
    """A paged server has one pool: what a sequence keeps goes to pages that nobody has."""
    from astc_kv_cuda import Q8Cache, Q8Evict
    page, block, keep = 64, 32, 150
    src, k, v = make(3, 2, 512, 64, fmt=fmt, block=block, page=page, spare=12, seed=4)
    used = set(src.block_table.flatten().tolist())
    free = torch.tensor([i for i in range(src.k.shape[0]) if i not in used][:9], dtype=torch.int32, device="cuda").view(3, 3)
    dst = Q8Cache(src.k, src.v, src.k_scales, src.v_scales, block_tokens=block, block_table=free)
    before = [t.clone() for t in (src.k.view(torch.int8), src.k_scales)]
    w = torch.rand(3, 2, 512, device="cuda")
    kept, lens, _ = Q8Evict(src, dst, w, torch.tensor([512, 100, 317], dtype=torch.int32, device="cuda"), keep=keep, sinks=3, recent=9).run()
    assert lens.tolist() == [keep, 100, keep]
    check_packed((k, v), dst, kept, lens.tolist())
    others = sorted(set(range(src.k.shape[0])) - set(free.flatten().tolist()))
    assert torch.equal(src.k.view(torch.int8)[others], before[0][others]) and torch.equal(src.k_scales[others], before[1][others])
    with pytest.raises(ValueError):
        Q8Evict(src, src, w, keep=keep)


def test_evict_between_slices_of_one_tensor(cuda):
    """The caches of two layers, K and V side by side, in one allocation; and slices that do overlap."""
    from astc_kv_cuda import Q8Cache, Q8Evict
    codes = torch.randint(-127, 128, (2, 2, 2, 3, 96, 64), device="cuda", dtype=torch.int8)  # batch, layer, K and V, ...
    scales = torch.rand(2, 2, 2, 3, 3, device="cuda")

    def cache(layer, t0, t1):
        c, s = codes[:, layer, :, :, t0:t1], scales[:, layer, :, :, t0 // 32:t1 // 32]
        return Q8Cache(c[:, 0], c[:, 1], s[:, 0], s[:, 1], block_tokens=32)
    w = torch.rand(2, 3, 96, device="cuda")
    for src, dst in ((cache(0, 0, 96), cache(1, 0, 96)), (cache(1, 0, 64), cache(1, 64, 96))):
        values = values_of(src)
        kept, lens, _ = Q8Evict(src, dst, w, keep=20).run()
        check_packed(values, dst, kept, lens.tolist())
    for src, dst in ((cache(0, 0, 96), cache(0, 64, 96)), (cache(1, 32, 96), cache(1, 0, 64))):
        with pytest.raises(ValueError):
            Q8Evict(src, dst, w, keep=20)


@pytest.mark.parametrize("paged", [False, True])
def test_no_sequences(cuda, paged):
    """A batch of none: empty results, no error."""
    from astc_kv_cuda import Q8Attention, Q8Cache, q8_evict, q8_restore, q8_store
    i32 = dict(dtype=torch.int32, device="cuda")

    def cache():
        paging = dict(block_table=torch.empty(0, 2, **i32), page_tokens=64, num_pages=4) if paged else {}
        return Q8Cache.zeros(0, 2, 128, 64, **paging)
    src, dst, none = cache(), cache(), torch.empty(0, **i32)
    x = torch.randn(0, 3, 2, 64, device="cuda")
    q8_store(src, x, x, none)
    assert q8_restore(src, none, 5)[0].shape == (0, 5, 2, 64)
    w = torch.empty(0, 2, 128, device="cuda")
    assert Q8Attention(torch.randn(0, 7, 8, 64, device="cuda"), src, none, weights=w, lse=True).run().shape == (0, 7, 8, 64)
    kept, lens, _ = q8_evict(src, dst, w, none, keep=10)
    assert kept.shape == (0, 2, 10) and lens.shape == (0,)


def test_no_queries(cuda):
    """A sum over no queries is 0, and adding it changes nothing."""
    from astc_kv_cuda import Q8Attention
    cache, _, _ = make(2, 3, 100, 64, seed=2)
    q = torch.randn(2, 0, 6, 64, device="cuda").bfloat16()
    w = torch.rand(2, 3, cache.max_tokens + 7, device="cuda")
    first = w.clone()
    assert Q8Attention(q, cache, weights=w).run().shape == (2, 0, 6, 64) and torch.equal(w, first)
    Q8Attention(q, cache, weights=w, accumulate=False).run()
    assert not w[:, :, :cache.max_tokens].any() and torch.equal(w[:, :, cache.max_tokens:], first[:, :, cache.max_tokens:])


def test_store_of_no_rows_anywhere(cuda):
    """A sequence that brings no rows stores nothing outside the cache, wherever its start is."""
    from astc_kv_cuda import Q8Cache, q8_store
    c = Q8Cache.zeros(4, 1, 64, 16, block_tokens=16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = Q8Cache(c.k, c.v, c.k_scales, c.v_scales, block_tokens=16, status=status)
    x = torch.ones(4, 8, 1, 16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    q8_store(cache, x, x, torch.tensor([-5, 64, 1 << 30, 3], **i32), torch.tensor([0, 0, -2, 1], **i32))
    assert int(status) == 0 and (cache.k[3, 0, 3] == 127).all() and not cache.k[:3].any()
    q8_store(cache, x, x, torch.tensor([-5, 64, 1 << 30, 3], **i32), torch.tensor([0, 0, 1, 1], **i32))
    assert int(status) == 1


def test_restore_where_an_eviction_of_empty_sequences_says(cuda):
    """A restore reads the lengths that the eviction before it wrote, also when there was nothing to pack."""
    from astc_kv_cuda import Q8Cache, Q8Evict, Q8Restore
    cache, _, _ = make(64, 2, 4096, 32, seed=5)
    dst = Q8Cache.zeros(64, 2, 64, 32, block_tokens=32)
    w = torch.rand(64, 2, 4096, device="cuda")
    lens = torch.zeros(64, dtype=torch.int32, device="cuda")
    evict = Q8Evict(cache, dst, w, lens, keep=32)
    restore = Q8Restore(dst, evict.lens, 1)
    dst.k[:, :, 0], dst.k[:, :, 32] = 1, 2
    dst.k_scales.fill_(1.0)
    for _ in range(200):
        evict.lens.fill_(32)
        evict.run()
        k, _ = restore.run()
        assert (k == 1).all()


@pytest.mark.parametrize("paged", [False, True])
def test_empty_cache_with_a_status(cuda, paged):
    from astc_kv_cuda import Q8Cache, q8_store
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    paging = dict(block_table=torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), page_tokens=32, num_pages=1) if paged else {}
    cache = Q8Cache.zeros(1, 1, 64, 32, block_tokens=32, status=status, **paging)
    x = torch.ones(1, 8, 1, 32, device="cuda")
    q8_store(cache, x, x, torch.full((1,), 4, dtype=torch.int32, device="cuda"))
    assert int(status) == 0
    q8_store(cache, x, x, torch.full((1,), 32 if paged else 60, dtype=torch.int32, device="cuda"))
    assert int(status) == (5 if paged else 1)
    with pytest.raises(ValueError):
        Q8Cache.zeros(1, 1, 64, 32, status=status.long())


def attention_off(cache, b, k, v, length, n, od):
    """Attention of random queries of every sequence over its whole cache, of which `b`'s last `length` tokens are k, v
    [H, length, D] and the rest is zeros: checks its outputs and weights."""
    from astc_kv_cuda import Q8Attention
    H, D, T, G = cache.kv_heads, cache.head_dim, cache.max_tokens, 4
    q = torch.randn(cache.batch, n, H * G, D, device="cuda").bfloat16()
    w = torch.zeros(cache.batch, H, T, device="cuda")
    out = Q8Attention(q, cache, out_dtype=od, weights=w).run()[b].double()
    qq = q[b].double().view(n, H, G, D).permute(1, 2, 0, 3)
    s = torch.einsum("hgnd,htd->hgnt", qq, k) * D ** -0.5
    A = float(torch.einsum("hgnd,htd->hgnt", qq.abs(), k.abs()).max()) * D ** -0.5
    hidden = torch.arange(length, device="cuda") > torch.arange(length - n, length, device="cuda").view(n, 1)
    e = s.masked_fill(hidden, float("-inf")).exp()
    p = e / (e.sum(-1, keepdim=True) + (T - length))  # every other token has score 0 and value 0
    ref = torch.einsum("hgnt,htd->nhgd", p, v).reshape(n, H * G, D)
    f, vmax = 2.0 ** -19 * A + 2.0 ** -18, float(v.abs().max())
    half = od != torch.float32
    assert ((out - ref).abs() <= vmax * (f + (2.0 ** -10 if half else 0.0)) + (2.0 ** -8 if half else 0.0) * ref.abs()).all()
    got = w[b, :, T - length:].double()
    assert ((got - p.sum((1, 2))).abs() <= p.sum((1, 2)) * f + 2.0 ** -22 * got + 1e-30).all()


def test_offsets_past_32_bits_of_one_piece(cuda):
    """The last sequence of more than 2^32 bytes of codes: store, restore, both attention kernels with weights, eviction."""
    from astc_kv_cuda import Q8Cache, q8_evict, q8_restore, q8_store
    B, H, T, D, n = 34, 8, 131072, 128, 300
    assert B * H * T * D > 1 << 32
    cache = Q8Cache.zeros(B, H, T, D, block_tokens=128)
    x, y = torch.randn(2, B, n, H, D, device="cuda").bfloat16()
    q8_store(cache, x, y, torch.full((B,), T - n, dtype=torch.int32, device="cuda"))
    back = q8_restore(cache, torch.full((B,), T - n, dtype=torch.int32, device="cuda"), n)
    for got, rows in zip(back, (x, y)):
        assert ((got - rows.float()).abs() <= rows.float().abs().amax((1, 2, 3), keepdim=True) / 127 * 0.51).all()
    k, v = (t[-1].double().transpose(0, 1) for t in back)
    attention_off(cache, B - 1, k, v, n, 4, torch.float32)
    attention_off(cache, B - 1, k, v, n, 16, torch.bfloat16)
    w = torch.zeros(B, H, T, device="cuda")
    w[-1, :, -n:] = torch.rand(H, n, device="cuda") + 1
    dst = Q8Cache.zeros(B, H, 128, D, block_tokens=128)
    kept, _, _ = q8_evict(cache, dst, w, keep=128)
    assert (kept[-1] >= T - n).all()
    for h in range(H):
        at = kept[-1, h].long() - (T - n)
        for got, rows in zip(values_of(dst), (k, v)):
            assert ((got[-1, h] - rows[h, at]).abs() <= rows[h, at].abs().max() / 127 * 0.51).all()


def test_offsets_past_32_bits_of_pages(cuda):
    """The last pages of a pool of more than 2^32 bytes: every call, and an eviction into other such pages."""
    from astc_kv_cuda import Q8Cache, q8_evict, q8_restore, q8_store
    pages, H, P, D, block, n = 17408, 8, 256, 128, 64, 1000
    assert pages * H * P * D > 1 << 32
    table = torch.tensor([[pages - 1, pages - 5, pages - 2, 3]], dtype=torch.int32, device="cuda")
    cache = Q8Cache.zeros(1, H, 4 * P, D, fmt="fp8", block_tokens=block, page_tokens=P, block_table=table, num_pages=pages)
    x, y = torch.randn(2, 1, n, H, D, device="cuda").bfloat16()
    q8_store(cache, x, y, torch.full((1,), 4 * P - n, dtype=torch.int32, device="cuda"))
    back = q8_restore(cache, torch.full((1,), 4 * P - n, dtype=torch.int32, device="cuda"), n)
    for got, rows in zip(back, (x, y)):
        assert ((got - rows.float()).abs() <= rows.float().abs() / 16 * 1.01 + rows.abs().max().float() / 448 * 2.0 ** -10).all()
    k, v = (t[0].double().transpose(0, 1) for t in back)
    attention_off(cache, 0, k, v, n, 4, torch.float32)
    attention_off(cache, 0, k, v, n, 200, torch.bfloat16)
    to = torch.tensor([[pages - 3, pages - 4]], dtype=torch.int32, device="cuda")
    dst = Q8Cache(cache.k, cache.v, cache.k_scales, cache.v_scales, block_tokens=block, block_table=to)
    w = torch.rand(1, H, 4 * P, device="cuda")
    w[:, :, :4 * P - n] = -1
    kept, lens, _ = q8_evict(cache, dst, w, keep=500)
    full = [torch.zeros(1, H, 4 * P, D, dtype=torch.float64, device="cuda") for _ in range(2)]
    for f, t in zip(full, (k, v)):
        f[0, :, 4 * P - n:] = t
    used = own_pages(dst)
    check_packed(full, used, kept, lens.tolist())


def own_pages(dst):
    """`dst`'s pages in a pool of their own, so that only they are looked at."""
    from astc_kv_cuda import Q8Cache
    at = dst.block_table.flatten().long()
    table = torch.arange(at.numel(), dtype=torch.int32, device="cuda").view(dst.block_table.shape)
    pool = [t.view(torch.int8)[at].view(t.dtype) for t in (dst.k, dst.v)] + [t[at] for t in (dst.k_scales, dst.v_scales)]
    return Q8Cache(*pool, block_tokens=dst.block_tokens, block_table=table)


@pytest.mark.parametrize("op", ["attention", "restore", "evict"])
def test_built_on_a_stream_of_its_own(cuda, op):
    """A call built on a side stream and run on the default one waits for the side stream's work on its memory."""
    build = small_calls()[op]
    want = [t.clone() for t in results(build().run())]
    side = torch.cuda.Stream()
    for _ in range(3):
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)
            junk = [torch.full_like(t, 77) for t in want for _ in range(3)]
            del junk
            call = build()
        got = results(call.run())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
