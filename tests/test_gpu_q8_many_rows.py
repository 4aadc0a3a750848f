"""Attention of many rows (query tokens x heads of a kv head) over the 8-bit
cache: the forms with 16-bit queries and outputs, whose kernel takes 33 rows
and more, in one tile of rows, in two that share them, and with wide heads.
Plain implementations and bounds are those of test_gpu_q8.py."""

import pytest
import torch

from test_gpu_q8 import check_attention, make, plain_attention

pytestmark = pytest.mark.gpu

# head_dim, query heads per kv head, query tokens: rows shared by two tiles, tiles of their own, several of them, wide heads.
SHAPES = [(64, 1, 40), (128, 4, 32), (128, 2, 100), (64, 3, 90), (128, 4, 150), (256, 1, 40), (240, 2, 90)]


def one_hot(fmt, D, G, n, T, size, sign, at, seed):
    """A cache and queries whose scores are `size` times numbers of order one, the one of token `at` far above the
    others. Returns also the score of `at` (scale 1)."""
    cache, k, v = make(1, 2, T, D, fmt=fmt, block=32, seed=seed)
    c = torch.zeros(k.shape, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(seed)
    low, high = (-96, 97) if sign > 0 else (64, 121)
    c[..., 0] = torch.randint(low // 8, high // 8, k.shape[:3], generator=g, device="cuda").float() * 8
    c[:, :, at, 0] = 120 if sign > 0 else 16
    cache.k.copy_(c.to(cache.k.dtype))  # multiples of 8: e4m3 holds them too
    cache.k_scales.fill_(1 / 128)
    q = torch.zeros(1, n, 2 * G, D, device="cuda")
    q[..., 0] = sign * size
    return cache, v, q, sign * size * float(c[0, 0, at, 0]) / 128


@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 14, 2.0 ** 17])
@pytest.mark.parametrize("D,G,n,T,od", [(D, G, n, n + 333, torch.bfloat16) for D, G, n in SHAPES] + [
    (64, 3, 1, 9000, torch.float32), (128, 4, 1, 5000, torch.float32), (128, 8, 1, 700, torch.float32),
    (128, 4, 5, 3000, torch.float32), (256, 2, 1, 6000, torch.float32), (128, 4, 20, 2000, torch.float32)])
def test_large_scores_in_pieces(cuda, D, G, n, T, od, size):
    """Rows whose tokens several CTAs divide: the pieces are divided by their sum, not by the log-sum-exp, whose last
    bit is worth 2^-24 of the scores. One token has all the weight; an output is its V row, off by the rounding of the
    weight (to fp16 with 16-bit outputs) and of the output."""
    from astc_kv_cuda import Q8Attention
    for at in (3, T - n):
        cache, v, q, score = one_hot("int8", D, G, n, T, size, 1, at, seed=n)
        lens = torch.full((1,), T, dtype=torch.int32, device="cuda")
        call = Q8Attention(q.bfloat16(), cache, lens, scale=1.0, out_dtype=od, lse=True)
        out = call.run().double().view(1, n, 2, G, D)
        want = v[:, :, at].view(1, 1, 2, 1, D).expand_as(out)
        off = 2.0 ** -18 + (2.0 ** -10 + 2.0 ** -8 if od == torch.bfloat16 else 0.0)
        assert ((out - want).abs() <= off * want.abs()).all()
        assert ((call.lse.double() - score).abs() <= 2.0 ** -20 * abs(score) + 2.0 ** -18).all()


@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 22, 2.0 ** 27, 2.0 ** 29, 2.0 ** 33, 2.0 ** 70, 2.0 ** 120])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("D,G,n", SHAPES)
def test_scores_of_any_magnitude(cuda, D, G, n, fmt, sign, size):
    """The softmax weight of one token is 1 (up to rounding it to fp16), whatever the size of the scores; tokens that
    are not seen do not count, even where every score is far below 0."""
    from astc_kv_cuda import Q8Attention
    T = n + 333
    for at in (3, T - n):
        cache, v, q, score = one_hot(fmt, D, G, n, T, size, sign, at, seed=n)
        lens = torch.full((1,), T, dtype=torch.int32, device="cuda")
        call = Q8Attention(q.bfloat16(), cache, lens, scale=1.0, out_dtype=torch.bfloat16, lse=True)
        out = call.run().double().view(1, n, 2, G, D)
        want = v[:, :, at].view(1, 1, 2, 1, D).expand_as(out)
        assert ((out - want).abs() <= (2.0 ** -10 + 2.0 ** -8 + 2.0 ** -18) * want.abs()).all()
        assert ((call.lse.double() - score).abs() <= 2.0 ** -20 * abs(score) + 2.0 ** -18).all()


@pytest.mark.parametrize("split", [16, 48, 64, 192, 512])
@pytest.mark.parametrize("D,G,n", SHAPES)
def test_splits_of_any_length(cuda, D, G, n, split):
    """split_tokens may be any multiple of 16; what lies between a split's end and the next step's is not a token."""
    cache, k, v = make(2, 2, n + 800, D, page=128 if D == 128 else 0, block=32, seed=D + n)
    q = torch.randn(2, n, 2 * G, D, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [n + 800, n + 77], out_dtype=torch.bfloat16, split=split)


@pytest.mark.parametrize("what", ["k_scales", "v_scales"])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("D,G,n,od", [(D, G, n, torch.bfloat16) for D, G, n in SHAPES] + [
    (64, 2, 4, torch.float32), (128, 4, 20, torch.float32), (128, 4, 4, torch.bfloat16), (256, 2, 50, torch.float32)])
def test_nan_scale_shows_where_it_is_seen(cuda, D, G, n, od, fmt, what):
    """A block with a NaN scale among the queries' own tokens: queries that see a token of it are NaN, queries that
    end before it, queries past q_lens and queries that see nothing are as without it."""
    from astc_kv_cuda import Q8Attention
    T, block = n + 256, 16
    cache, k, v = make(3, 2, T, D, fmt=fmt, block=block, seed=n + D)
    lens, q_lens = [T, T - 5, n // 2], [n, n - 3, n]
    q = torch.randn(3, n, 2 * G, D, device="cuda").bfloat16()
    ref, lse, _, A, vmax = plain_attention(q, k, v, lens, q_lens)
    first = []  # of the block's tokens
    for b in range(3):
        at = (lens[b] - 2) // block
        getattr(cache, what)[b, :, at] = float("nan")
        first.append(at * block)
    i32 = dict(dtype=torch.int32, device="cuda")
    call = Q8Attention(q, cache, torch.tensor(lens, **i32), q_lens=torch.tensor(q_lens, **i32), out_dtype=od, lse=True)
    out = call.run().double()
    f = 2.0 ** -19 * A + 2.0 ** -18
    tol = vmax * (f + (0.0 if od == torch.float32 else 2.0 ** -10)) + (0.0 if od == torch.float32 else 2.0 ** -8) * ref.abs() + 1e-30
    for b in range(3):
        for i in range(n):
            end = lens[b] - q_lens[b] + i + 1 if i < q_lens[b] else 0  # tokens that the query sees
            if end > first[b]:
                assert out[b, i].isnan().all() and call.lse[b, i].isnan().all(), (b, i)
            else:
                assert ((out[b, i] - ref[b, i]).abs() <= tol[b, i]).all(), (b, i)
                assert torch.equal(call.lse[b, i].isinf(), lse[b, i].isinf()) and not call.lse[b, i].isnan().any(), (b, i)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("D,G,n,od", [(128, 4, 40, torch.bfloat16), (256, 1, 40, torch.bfloat16), (128, 4, 6, torch.float32),
                                      (64, 1, 20, torch.float32)])
def test_stored_nan_stays_with_its_block(cuda, D, G, n, od, fmt, bad):
    """Queries that end before the block of a row that is not finite are as without it, after a store and after an eviction."""
    from astc_kv_cuda import Q8Attention, Q8Cache, Q8Evict, q8_store
    T, block = 192, 16
    at = T - 3
    x = [torch.randn(1, T, 2, D, device="cuda") for _ in range(2)]
    caches = []
    for value in (0.0, bad):
        for y in x:
            y[0, at, :, 5] = value
        c = Q8Cache.zeros(1, 2, T, D, fmt=fmt, block_tokens=block)
        caches.append(q8_store(c, *x, torch.zeros(1, dtype=torch.int32, device="cuda")))
    w = torch.zeros(1, 2, T, device="cuda")
    small = []
    for c in caches:
        small.append(Q8Cache.zeros(1, 2, T - block, D, fmt=fmt, block_tokens=block))
        Q8Evict(c, small[-1], w, keep=T - block, recent=2 * block).run()
    q = torch.randn(1, n, 2 * G, D, device="cuda").bfloat16()
    for (good, poor), length in ((caches, T), (small, T - block)):
        codes = [t.view(torch.uint8) for t in (poor.k, poor.v)]
        assert fmt == "int8" or not any(((t & 127) == 127).any() for t in codes)
        clean, out = (Q8Attention(q, c, out_dtype=od).run() for c in (good, poor))
        sees = length - n + torch.arange(n, device="cuda") + 1 > length - block
        assert out[0, sees].isnan().all() and torch.equal(out[0, ~sees], clean[0, ~sees])


@pytest.mark.parametrize("size", [2.0 ** 18, 2.0 ** 22, 2.0 ** 23, 2.0 ** 24, 2.0 ** 25, 2.0 ** 26, 2.0 ** 27])
@pytest.mark.parametrize("n,od", [(1, torch.float32), (1, torch.bfloat16), (2, torch.float32), (40, torch.bfloat16)])
def test_large_scores_that_rise(cuda, n, od, size):
    """Scores near `size` that rise by some 5 to 12 natural units every 64 tokens, where fp32 has few bits or none for the
    differences: an output stays among the values that it averages."""
    from astc_kv_cuda import Q8Attention
    T, D, G = 1024, 64, 8
    cache, _, v = make(8, 1, T, D, block=32, seed=1, spread=0.0)
    cache.k.zero_()
    cache.k[..., 0] = 64
    cache.k[..., 1] = (torch.arange(T, device="cuda") // 64).to(torch.int8)
    cache.k_scales.fill_(1 / 64)
    q = torch.zeros(8, n, G, D, device="cuda")
    q[..., 0] = size
    q[..., 1] = 64 * torch.linspace(5.0, 12.0, 64, device="cuda").view(8, 1, G)
    lens = torch.full((8,), T, dtype=torch.int32, device="cuda")
    # Splits of all tokens, so that one warp goes through the rise.
    call = Q8Attention(q.bfloat16() if n == 40 else q, cache, lens, scale=1.0, out_dtype=od, lse=True, split_tokens=T)
    out = call.run().double()
    top = v.abs().amax()
    assert (out.abs() <= top * (1 + 2.0 ** -7)).all()  # a NaN or an infinity is not
    score = q[..., 0].double() + q[..., 1].double() / 64 * (T // 64 - 1)
    assert ((call.lse.double() - score).abs() <= 2.0 ** -19 * score + 16).all()


@pytest.mark.parametrize("D,G,n", SHAPES)
def test_bad_table_entries_read_as_zeros(cuda, D, G, n):
    from astc_kv_cuda import Q8Cache
    made, k, v = make(2, 2, 512, D, page=128, block=32, seed=10)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = Q8Cache(made.k, made.v, made.k_scales, made.v_scales, block_tokens=32, block_table=made.block_table, status=status)
    cache.block_table[0, 1], cache.block_table[1, 2] = 99999, -1
    for x in (k, v):
        x[0, :, 128:256] = 0
        x[1, :, 256:384] = 0
    q = torch.randn(2, n, 2 * G, D, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [512, 300], out_dtype=torch.bfloat16)
    assert int(status) == 5


@pytest.mark.parametrize("D,G,n", SHAPES)
def test_runs_repeat_bit_for_bit(cuda, D, G, n):
    """Outputs, log-sum-exps and token weights, which other kernels compute from them."""
    from astc_kv_cuda import Q8Attention
    cache, _, _ = make(3, 2, 3000, D, page=256, block=64, seed=12)
    q = torch.randn(3, n, 2 * G, D, device="cuda").half()
    lens = torch.tensor([3000, 1234, 177], dtype=torch.int32, device="cuda")
    w = torch.zeros(3, 2, cache.max_tokens, device="cuda")
    call = Q8Attention(q, cache, lens, weights=w, accumulate=False, out_dtype=torch.float16, lse=True)
    a = call.run().clone(), call.lse.clone(), w.clone()
    for _ in range(5):
        call.run()
        assert torch.equal(call.out, a[0]) and torch.equal(call.lse, a[1]) and torch.equal(w, a[2])


@pytest.mark.parametrize("D,G,n", SHAPES)
def test_in_a_graph(cuda, D, G, n):
    """Store, attention with weights and eviction in one graph, which follows the lengths."""
    from astc_kv_cuda import Q8Attention, Q8Cache, Q8Evict, Q8Store
    i32 = dict(dtype=torch.int32, device="cuda")
    T, keep = 1024, 96
    lens, start = torch.zeros(2, **i32), torch.zeros(2, **i32)
    cache, dst = Q8Cache.zeros(2, 2, T, D), Q8Cache.zeros(2, 2, 128, D)
    x, y = (torch.zeros(2, n, 2, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q = torch.zeros(2, n, 2 * G, D, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(2, 2, T, device="cuda")
    calls = [Q8Store(cache, x, y, start), Q8Attention(q, cache, lens, out_dtype=torch.bfloat16, weights=w),
             Q8Evict(cache, dst, w, lens, keep=keep, recent=8)]

    def run():
        return [t.clone() for c in calls for t in (lambda r: r if isinstance(r, tuple) else (r,))(c.run()) if torch.is_tensor(t)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    fresh = [t.clone() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales, w)]
    results = []
    for replay in (True, False):
        for t, f in zip((cache.k, cache.v, cache.k_scales, cache.v_scales, w), fresh):
            t.copy_(f)
        g = torch.Generator(device="cuda").manual_seed(3)
        for at in (0, n, 2 * n):
            start.copy_(torch.tensor([at, at // 2], **i32))
            lens.copy_(start + n)
            for t in (x, y, q):
                t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
            if replay:
                graph.replay()
                results.append([t.clone() for t in got])
            else:
                assert all(torch.equal(a, b) for a, b in zip(results.pop(0), run()))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("D,G,n,T", [(64, 3, 1, 65536), (128, 4, 1, 65536), (128, 8, 1, 30010), (128, 4, 4, 40000), (256, 2, 1, 65536),
                                     (256, 8, 3, 30010), (64, 9, 1, 1025), (64, 1, 1, 4099)])
def test_long_sums_do_not_shrink(cuda, D, G, n, T, fmt):
    """Outputs are means of equal values, summed by one warp group over all tokens: what is lost is what the sums lose. 32
    sums that truncate at 2^-23, on the average at half of what they come to, make 2^-19; the parts of the softmax
    weights (2^-22), the exponentials (2^-22) and the sums to nearest the rest of 2^-18."""
    from astc_kv_cuda import Q8Attention
    cache, _, _ = make(2, 1, T, D, fmt=fmt, block=32, seed=T)
    cache.v.copy_(torch.full(cache.v.shape, 104.0, device="cuda").to(cache.v.dtype))
    cache.v_scales.fill_(1 / 96)
    q = torch.randn(2, n, G, D, device="cuda").bfloat16()
    lens = torch.tensor([T, T - 777], dtype=torch.int32, device="cuda")
    out = Q8Attention(q, cache, lens, scale=0.3 * D ** -0.5, split_tokens=(T + 15) // 16 * 16).run().double()
    value = float(torch.tensor(1 / 96)) * 104
    assert ((out - value).abs() <= 2.0 ** -18 * value).all()


@pytest.mark.parametrize("n,H", [(16, 4), (100, 2)])
def test_long_sums_of_fp16_outputs(cuda, n, H):
    """Row tiles for 148 SMs, so that nothing but length asks for splits. Outputs are 64 known values, each rounded to
    fp16, 2^-11 at most and at random: their mean is off by 2^-14.8, one standard deviation. Sums that lose 2^-27.3 of
    themselves with every token, over 16384 of them, lose 2^-13.3."""
    from astc_kv_cuda import Q8Attention, Q8Cache
    B, G, T, D = 37, 4, 131072, 64
    cache = Q8Cache.zeros(B, H, T, D, block_tokens=128)
    cache.k.random_(-100, 101)
    cache.v.copy_(torch.arange(64, 128, device="cuda").to(torch.int8).expand(cache.v.shape))
    cache.k_scales.fill_(1 / 100)
    cache.v_scales.fill_(1 / 96)
    q = torch.randn(B, n, H * G, D, device="cuda").half()
    out = Q8Attention(q, cache, out_dtype=torch.float16).run().double()
    value = float(torch.tensor(1 / 96)) * torch.arange(64, 128, device="cuda").double()
    off = (out / value - 1).mean(-1)
    assert (off.abs() <= 2.0 ** -12).all()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("D", [144, 208, 256])
@pytest.mark.parametrize("n", [8, 9, 16, 17, 24, 32])
def test_wide_heads_of_few_rows(cuda, D, n, fmt):
    cache, k, v = make(2, 2, 500, D, fmt=fmt, block=32, seed=n)
    q = torch.randn(2, n, 2, D, device="cuda").half()
    check_attention(cache, k, v, q, [500, 130], [n, n // 2], out_dtype=torch.float16)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), 3e38])
@pytest.mark.parametrize("D,G,n,od", [(D, G, n, torch.bfloat16) for D, G, n in SHAPES] + [
    (64, 2, 4, torch.float32), (128, 4, 20, torch.float32), (128, 4, 4, torch.bfloat16)])
def test_queries_past_their_count_are_not_looked_at(cuda, D, G, n, od, value):
    """What lies past q_lens (and in sequences without queries) reaches no output and no weight."""
    from astc_kv_cuda import Q8Attention
    cache, _, _ = make(3, 2, 300, D, block=32, seed=n)
    i32 = dict(dtype=torch.int32, device="cuda")
    lens, q_lens = torch.tensor([300, 200, 250], **i32), torch.tensor([n - 1, n // 2, 0], **i32)
    q = torch.randn(3, n, 2 * G, D, device="cuda").bfloat16()
    results = []
    for fill in (0.0, value):
        for b, m in enumerate(q_lens.tolist()):
            q[b, m:] = fill
        w = torch.ones(3, 2, cache.max_tokens, device="cuda")
        call = Q8Attention(q, cache, lens, q_lens=q_lens, out_dtype=od, lse=True, weights=w)
        results.append((call.run(), call.lse, w))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    for b, m in enumerate(q_lens.tolist()):
        assert not results[1][0][b, m:].any() and (results[1][1][b, m:] == float("-inf")).all()
