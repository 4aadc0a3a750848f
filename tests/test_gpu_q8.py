"""The 8-bit KV cache on the GPU against plain implementations in 64 bits.

Bounds. A stored value is off by at most half a step of its format: scale / 2
for int8; for e4m3 |x| / 16 (three bits after the leading one) or, below the
smallest normal code, scale / 2^10. A block that grows adds one more rounding
to the rows it held. The fp32 products around it (amax * (1/M), x * (1/scale))
are off by a few 2^-24, far below 2^-10 of a step.

Attention: a score is a sum of D <= 256 products in fp32, in at most 16
accumulating steps that may truncate, so it is off by at most 2^-20 A with A
the largest sum of |scale q k| of a row; that makes every softmax weight off
by a factor of at most 1 +- 2^-19 A, and 2^-18 covers exp2, the running sums
and V's part. An output is a weighted mean of V's rows: the bound is
max |V| (2^-19 A + 2^-18), plus 2^-10 max |V| where the softmax weights are
rounded to fp16 (16-bit outputs), plus half an ulp of the output's type. A
token's weight is a sum of softmax weights: the same factors of itself.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

MOST = {"int8": 127.0, "fp8": 448.0}


def make(B, H, T, D, *, fmt="int8", block=32, page=0, seed=0, spare=0, spread=0.5):
    """A cache of T tokens per sequence filled with random codes and scales, in
    one piece or in shuffled pages; and its K and V [B, H, T, D] in 64 bits."""
    from astc_kv_cuda import Q8Cache
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    room = -(-T // (page or block)) * (page or block)
    per = room // (page or room)
    n = B * per + spare
    shape = (n, H, page or room, D)
    table = torch.randperm(n, generator=g, device="cuda")[:B * per].view(B, per).to(torch.int32) if page else None
    codes, scales, values = [], [], []
    for side in range(2):
        x = torch.randn(shape, generator=g, device="cuda") * MOST[fmt] / 4
        c = x.clamp(-MOST[fmt], MOST[fmt]).round().to(dt) if fmt == "int8" else x.clamp(-448, 448).to(dt)
        s = torch.exp(spread * torch.randn(n, H, shape[2] // block, generator=g, device="cuda")) * 4 / MOST[fmt]
        v = c.double() * s.double().repeat_interleave(block, 2)[..., None]
        if page:
            v = v[table.long()].transpose(1, 2).reshape(B, H, room, D)
        codes.append(c)
        scales.append(s)
        values.append(v)
    cache = Q8Cache(codes[0], codes[1], scales[0], scales[1], block_tokens=block, block_table=table, max_tokens=room)
    return cache, values[0], values[1]


def plain_attention(q, k, v, lens, q_lens, causal=True, scale=None):
    """out [B, n, Hq, D], lse [B, n, Hq], weights [B, H, T], A and max |V|, in 64 bits."""
    B, n, Hq, D = q.shape
    H, T = k.shape[1], k.shape[2]
    G = Hq // H
    scale = scale or D ** -0.5
    out = torch.zeros(B, n, Hq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, n, Hq), -math.inf, dtype=torch.float64, device=q.device)
    w = torch.zeros(B, H, T, dtype=torch.float64, device=q.device)
    A = vmax = 0.0
    for b in range(B):
        ln, qn = min(max(lens[b], 0), T), min(max(q_lens[b], 0), n)
        for i in range(qn):
            end = max(ln - qn + i + 1, 0) if causal else ln
            if end == 0:
                continue
            for h in range(H):
                kk, vv = k[b, h, :end], v[b, h, :end]
                qq = q[b, i, h * G:(h + 1) * G].double()
                s = qq @ kk.T * scale
                A = max(A, float((qq.abs() @ kk.abs().T).max()) * scale)
                vmax = max(vmax, float(vv.abs().max()))
                lse[b, i, h * G:(h + 1) * G] = torch.logsumexp(s, 1)
                p = torch.softmax(s, 1)
                out[b, i, h * G:(h + 1) * G] = p @ vv
                w[b, h, :end] += p.sum(0)
    return out, lse, w, A, vmax


def check_attention(cache, k, v, q, lens, q_lens=None, *, out_dtype=torch.float32, weights=True, accumulate=True, causal=True,
                    scale=0.0, split=0, lens_none=False):
    from astc_kv_cuda import Q8Attention
    B = cache.batch
    rows = q if q.dim() == 4 else q.unsqueeze(1)
    n = rows.shape[1]
    lt = None if lens_none else torch.tensor(lens, dtype=torch.int32, device="cuda")
    qt = torch.tensor(q_lens, dtype=torch.int32, device="cuda") if q_lens is not None else None
    first = torch.rand(B, cache.kv_heads, cache.max_tokens, device="cuda") if weights else None
    w = first.clone() if weights else None
    call = Q8Attention(q, cache, lt, q_lens=qt, causal=causal, scale=scale, out_dtype=out_dtype, lse=True, weights=w,
                       accumulate=accumulate, split_tokens=split)
    call.out.fill_(float("nan"))
    call.workspace.view(torch.uint8).fill_(255)
    out = call.run().double().view(rows.shape)
    torch.cuda.synchronize()
    ref, lse, wref, A, vmax = plain_attention(rows, k, v, lens, q_lens or [n] * B, causal, scale or None)
    f = 2.0 ** -19 * A + 2.0 ** -18
    half_ulp = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[out_dtype]
    tol = vmax * (f + (2.0 ** -10 if out_dtype != torch.float32 else 0.0)) + half_ulp * ref.abs() + 1e-30
    bad = ~((out - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outputs off, worst {float((out - ref).abs().max()):.3e}, bound {float(tol.max()):.3e}"
    got = call.lse.double()
    assert torch.equal(torch.isinf(got), torch.isinf(lse)) and not torch.isnan(got).any()
    fin = ~torch.isinf(lse)
    assert ((got - lse)[fin].abs() <= f + 2.0 ** -22 * lse[fin].abs()).all()
    if weights:
        pos = torch.arange(cache.max_tokens, device="cuda")
        inside = pos.view(1, 1, -1) < torch.tensor(lens, device="cuda").clamp(0, cache.max_tokens).view(B, 1, 1)
        want = torch.where(inside, wref + (first.double() if accumulate else 0.0), first.double() if accumulate else torch.zeros_like(wref))
        assert ((w.double() - want).abs() <= wref * f + 2.0 ** -22 * want + 1e-30).all()
    return call


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("G,H,D", [(3, 3, 64), (4, 2, 128), (8, 1, 128), (1, 4, 64), (16, 1, 128), (3, 2, 80), (4, 1, 96), (2, 2, 256),
                                   (1, 2, 16), (20, 1, 48), (5, 1, 240)])
def test_one_token_head_layouts(cuda, fmt, G, H, D):
    cache, k, v = make(2, H, 300, D, fmt=fmt, seed=G * D)
    q = torch.randn(2, G * H, D, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [300, 177])


@pytest.mark.parametrize("T", [1, 2, 7, 15, 16, 17, 31, 33, 64, 127, 129, 255, 257, 391, 1025])
def test_one_token_lengths(cuda, T):
    cache, k, v = make(3, 2, T + 40, 64, block=16, seed=T)
    q = torch.randn(3, 6, 64, device="cuda").half()
    check_attention(cache, k, v, q, [T, max(T - 1, 0), 0])


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_pages(cuda, block, fmt):
    cache, k, v = make(4, 2, 1024, 128, fmt=fmt, block=block, page=256, spare=5, seed=block)
    q = torch.randn(4, 8, 128, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [1024, 1, 255, 513])
    check_attention(cache, k, v, torch.randn(4, 37, 8, 128, device="cuda").bfloat16(), [1024, 12, 255, 513], [37, 12, 20, 1],
                    out_dtype=torch.bfloat16)


@pytest.mark.parametrize("qd", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("od", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_types(cuda, qd, od, n):
    cache, k, v = make(2, 2, 200, 128, seed=n)
    q = torch.randn(2, n, 8, 128, device="cuda").to(qd)
    check_attention(cache, k, v, q, [200, 131], out_dtype=od)


@pytest.mark.parametrize("n,T,q_lens,lens", [
    (2, 64, [2, 1], [64, 1]), (5, 130, [5, 3], [130, 3]), (5, 130, [0, 5], [70, 5]), (17, 257, [17, 9], [257, 200]),
    (33, 96, [33, 33], [96, 33]), (64, 64, [64, 1], [64, 64]), (100, 300, [100, 77], [300, 77]), (129, 150, [129, 128], [150, 150]),
    (260, 700, [260, 1], [700, 333]),
    (6, 64, [6, 6], [3, 0]),  # fewer cached tokens than queries: the first queries see nothing
])
@pytest.mark.parametrize("D,G", [(64, 3), (128, 4)])
@pytest.mark.parametrize("od", [torch.float32, torch.bfloat16])
def test_many_tokens(cuda, n, T, q_lens, lens, D, G, od):
    cache, k, v = make(2, 2, T, D, fmt="fp8" if D == 64 else "int8", block=16, seed=n + T)
    q = torch.randn(2, n, 2 * G, D, device="cuda").bfloat16()
    check_attention(cache, k, v, q, lens, q_lens, out_dtype=od)


@pytest.mark.parametrize("D,G,n,T", [(256, 4, 9, 40), (256, 8, 33, 300), (240, 2, 64, 129), (144, 1, 200, 517), (256, 1, 33, 33)])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_many_tokens_of_wide_heads(cuda, D, G, n, T, fmt):
    cache, k, v = make(2, 1, T, D, fmt=fmt, block=16, seed=D + n)
    q = torch.randn(2, n, G, D, device="cuda").half()
    check_attention(cache, k, v, q, [T, max(T // 2, n)], [n, n // 2 + 1], out_dtype=torch.float16)


@pytest.mark.parametrize("page,block", [(48, 16), (96, 32), (16, 16), (640, 128)])
@pytest.mark.parametrize("n", [1, 9, 70])
@pytest.mark.parametrize("D", [128, 256])
def test_page_sizes_that_are_no_powers_of_two(cuda, page, block, n, D):
    cache, k, v = make(2, 2, 1000, D, block=block, page=page, spare=3, seed=page + n)
    q = torch.randn(2, n, 8, D, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [1000, 333], out_dtype=torch.bfloat16)
    check_attention(cache, k, v, q, [997, 150])


@pytest.mark.parametrize("n,od", [(1, torch.float32), (3, torch.float32), (20, torch.bfloat16)])
def test_many_sequences(cuda, n, od):
    """More sequences than a CTA has threads, many of them empty."""
    B = 300
    cache, k, v = make(B, 1, 200, 64, block=16, seed=n)
    q = torch.randn(B, n, 2, 64, device="cuda").bfloat16()
    r = np.random.default_rng(n)
    lens = [int(x) if x % 3 else 0 for x in r.integers(0, 201, B)]
    q_lens = [int(x) for x in r.integers(0, n + 1, B)]
    check_attention(cache, k, v, q, lens, q_lens, out_dtype=od)
    check_attention(cache, k, v, q, [0] * B, q_lens, out_dtype=od, accumulate=False)


@pytest.mark.parametrize("T,lens", [(4096, [4096, 1]), (4000, [63, 0]), (700, [700, 449])])
@pytest.mark.parametrize("G", [1, 4, 8])
def test_one_token_of_few_heads(cuda, T, lens, G):
    cache, k, v = make(2, 2, T, 128, fmt="fp8", block=64, seed=T + G)
    q = torch.randn(2, 2 * G, 128, device="cuda")
    check_attention(cache, k, v, q, lens)
    check_attention(cache, k, v, q.half(), lens, out_dtype=torch.float16, accumulate=False)


@pytest.mark.parametrize("n", [1, 4, 50])
def test_not_causal_and_scale(cuda, n):
    cache, k, v = make(2, 1, 333, 64, seed=3)
    q = torch.randn(2, n, 5, 64, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [333, 100], causal=False, scale=0.37)
    check_attention(cache, k, v, q, [333, 0], causal=False, out_dtype=torch.float16, accumulate=False)


@pytest.mark.parametrize("split", [16, 48, 64, 1024])
def test_splits_agree(cuda, split):
    cache, k, v = make(2, 2, 1000, 128, page=128, seed=9)
    q = torch.randn(2, 8, 128, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [1000, 500], split=split)


def test_lens_none_and_long(cuda):
    cache, k, v = make(1, 2, 20000, 64, fmt="fp8", block=128, seed=4)
    q = torch.randn(1, 6, 64, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [cache.max_tokens], lens_none=True)


@pytest.mark.parametrize("n", [1, 30])
def test_scores_and_scales_of_any_size(cuda, n):
    """Peaked softmax (scores of hundreds), V scales over twelve decades, blocks of zeros."""
    from astc_kv_cuda import Q8Cache
    a, k, _ = make(2, 1, 640, 128, block=32, seed=5)
    b, _, v = make(2, 1, 640, 128, block=32, seed=5, spread=4.0)
    cache = Q8Cache(a.k, b.v, a.k_scales, b.v_scales, block_tokens=32)
    for c, s, x in ((cache.k, cache.k_scales, k), (cache.v, cache.v_scales, v)):
        s[:, :, 3] = 0
        x.view(2, 1, -1, 32, 128)[:, :, 3] = 0
        c[:, :, 5 * 32:6 * 32] = 0
        x.view(2, 1, -1, 32, 128)[:, :, 5] = 0
    q = torch.randn(2, n, 4, 128, device="cuda") * 30
    check_attention(cache, k, v, q, [640, 333])
    q = torch.randn(2, n, 4, 128, device="cuda") * 1e-3
    check_attention(cache, k, v, q.half(), [640, 333], out_dtype=torch.float16)


def test_large_and_tiny_queries(cuda):
    """fp32 queries whose values no 16-bit type holds."""
    cache, k, v = make(1, 1, 100, 64, seed=6)
    for f in (1e-20, 1e15):
        q = torch.randn(1, 2, 64, device="cuda") * f
        check_attention(cache, k, v, q, [100], scale=0.1 / f)
    q = torch.randn(1, 40, 2, 64, device="cuda") * 1e30
    check_attention(cache, k, v, q, [100], scale=1e-31)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("n", [1, 5, 64])
def test_what_lies_past_the_length_is_not_read_into_results(cuda, fmt, n):
    cache, k, v = make(2, 2, 256, 64, fmt=fmt, block=32, seed=7)
    lens = [n + 100, n + 64]
    for b in range(2):
        for c, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
            c.view(torch.int8)[b, :, lens[b]:] = 127  # e4m3: NaN
            s[b, :, -(-lens[b] // 32):] = float("nan") if b else float("inf")
    q = torch.randn(2, n, 4, 64, device="cuda").bfloat16()
    check_attention(cache, k, v, q, lens, out_dtype=torch.float32)
    check_attention(cache, k, v, q, lens, out_dtype=torch.bfloat16)


@pytest.mark.parametrize("n", [1, 20])
def test_nan_shows(cuda, n):
    from astc_kv_cuda import q8_attention
    cache, _, _ = make(2, 1, 96, 64, block=32, seed=8)
    cache.v_scales[0, 0, 1] = float("nan")
    q = torch.randn(2, n, 2, 64, device="cuda").bfloat16()
    out = q8_attention(q, cache, causal=False)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("n", [1, 24])
def test_bad_table_entries_read_as_zeros(cuda, n):
    cache, k, v = make(2, 2, 512, 64, page=128, block=32, seed=10)
    cache.status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache._c.status_dev = cache.status.data_ptr()
    cache.block_table[0, 1], cache.block_table[1, 2] = 99999, -1
    for x in (k, v):
        x[0, :, 128:256] = 0
        x[1, :, 256:384] = 0
    q = torch.randn(2, n, 4, 64, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [512, 300])
    assert int(cache.status) == 5


@pytest.mark.parametrize("n", [1, 40])
def test_strided_queries_and_caches(cuda, n):
    """Queries inside a fused projection; codes stored token-major ([B, T, H, D])."""
    from astc_kv_cuda import Q8Cache
    base, k, v = make(2, 3, 160, 64, block=32, seed=11)
    codes = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in (base.k, base.v)]
    pad = [torch.full((2, 160, 3, 96), 77, dtype=torch.int8, device="cuda")[..., 16:80].transpose(1, 2) for _ in range(2)]
    for p, c in zip(pad, codes):
        p.copy_(c)
    for kk, vv in ((codes[0], codes[1]), (pad[0], pad[1])):
        cache = Q8Cache(kk, vv, base.k_scales, base.v_scales, block_tokens=32)
        qkv = torch.randn(2, n, 9 + 2 * 3, 64, device="cuda").bfloat16()
        check_attention(cache, k, v, qkv[:, :, :9], [160, 99])
        q = torch.randn(2, n, 9, 72, device="cuda")[..., 1:65].half()
        odd = torch.empty(2, n, 9, 67, dtype=torch.float16, device="cuda")[..., 3:]  # rows on odd elements
        odd.copy_(q)
        check_attention(cache, k, v, odd, [160, 99], out_dtype=torch.float16)


@pytest.mark.parametrize("n", [1, 64])
def test_runs_repeat_bit_for_bit(cuda, n):
    from astc_kv_cuda import Q8Attention
    cache, _, _ = make(3, 2, 3000, 128, page=256, block=64, seed=12)
    q = torch.randn(3, n, 8, 128, device="cuda").bfloat16()
    lens = torch.tensor([3000, 1234, 77], dtype=torch.int32, device="cuda")
    w = torch.zeros(3, 2, cache.max_tokens, device="cuda")
    call = Q8Attention(q, cache, lens, weights=w, accumulate=False)
    a = call.run().clone(), w.clone()
    for _ in range(5):
        call.run()
        assert torch.equal(call.out, a[0]) and torch.equal(w, a[1])


def test_offsets_past_32_bits(cuda):
    """A cache of more than 2^32 bytes of codes: its last sequence and page."""
    from astc_kv_cuda import Q8Cache, q8_attention, q8_restore
    B, H, T, D = 34, 8, 131072, 128
    assert B * H * T * D > 1 << 32
    k = torch.zeros(B, H, T, D, dtype=torch.int8, device="cuda")
    v = torch.zeros_like(k)
    s = torch.ones(B, H, T // 128, device="cuda") / 64
    g = torch.Generator(device="cuda").manual_seed(1)
    for x in (k, v):
        x[-1, -1, -300:] = torch.randint(-127, 128, (300, D), generator=g, device="cuda", dtype=torch.int8)
    cache = Q8Cache(k, v, s, s.clone(), block_tokens=128)
    q = torch.randn(B, H, D, device="cuda").bfloat16()
    out = q8_attention(q, cache)[-1, -1].double()
    sc = k[-1, -1].double() @ q[-1, -1].double() / 64 / D ** 0.5
    ref = torch.softmax(sc, 0) @ (v[-1, -1].double() / 64)
    A = float((k[-1, -1].double().abs() @ q[-1, -1].double().abs()).max() / 64 / D ** 0.5)
    assert ((out - ref).abs() <= 2 * (2.0 ** -19 * A + 2.0 ** -18)).all()
    kk, _ = q8_restore(cache, torch.full((B,), T - 5, dtype=torch.int32, device="cuda"), 8)
    assert torch.equal(kk[-1, :5, -1], k[-1, -1, -5:].float() / 64) and not kk[:, 5:].any()


# ---------------------------------------------------------- store and restore

def values_of(cache):
    """K and V [B, H, T, D] of a cache, by indexing, in 64 bits."""
    out = []
    for c, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        v = c.double() * s.double().repeat_interleave(cache.block_tokens, 2)[:, :, :c.shape[2], None]
        if cache.block_table is not None:
            v = v[cache.block_table.long()].transpose(1, 2)
            v = v.reshape(cache.batch, cache.kv_heads, -1, cache.head_dim)
        out.append(v)
    return out


def half_step(x, scale, fmt):
    return scale * (0.5 + 2.0 ** -10) if fmt == "int8" else torch.maximum(x.abs() / 16, scale * 2.0 ** -10) * (1 + 2.0 ** -10)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("D", [16, 64, 80, 128, 256])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_store_in_steps(cuda, fmt, block, D, dt):
    """Tokens arrive in pieces of uneven length whose size grows, so that begun blocks need larger scales."""
    from astc_kv_cuda import Q8Cache, q8_restore, q8_store
    B, H, T = 2, 3, 300
    cache = Q8Cache.zeros(B, H, T, D, fmt=fmt, block_tokens=block)
    g = torch.Generator(device="cuda").manual_seed(block + D)
    x = [(torch.randn(B, T, H, D, generator=g, device="cuda") * torch.exp(torch.randn(B, T, 1, 1, generator=g, device="cuda"))).to(dt)
         for _ in range(2)]
    at, grown = [0, 0], torch.zeros(B, 2, H, T, dtype=torch.int64, device="cuda")
    before = [s.clone() for s in (cache.k_scales, cache.v_scales)]
    for n in (1, 1, 5, 40, 1, 100, 17, 64, 200):
        counts = [min(n, T - at[0]), min(max(n - 3, 0), T - at[1])]
        start = torch.tensor(at, dtype=torch.int32, device="cuda")
        rows = [torch.zeros(B, n, H, D, dtype=dt, device="cuda") for _ in x]
        for b in range(B):
            for r, full in zip(rows, x):
                r[b, :counts[b]] = full[b, at[b]:at[b] + counts[b]]
                r[b, counts[b]:] = float("nan")  # not read
        q8_store(cache, rows[0], rows[1], start, torch.tensor(counts, dtype=torch.int32, device="cuda"))
        for j, s in enumerate((cache.k_scales, cache.v_scales)):
            for b in range(B):
                blk = at[b] // block
                if at[b] % block and counts[b]:
                    more = (s[b, :, blk] > before[j][b, :, blk]).long()
                    grown[b, j, :, blk * block:at[b]] += more[:, None]
            before[j] = s.clone()
        at = [a + c for a, c in zip(at, counts)]
    assert at[0] == T
    for j, (got, s) in enumerate(zip(values_of(cache), (cache.k_scales, cache.v_scales))):
        scale = s.double().repeat_interleave(block, 2)[:, :, :T, None]
        want = x[j].double().transpose(1, 2)
        for b in range(B):
            w, sc = want[b, :, :at[b]], scale[b, :, :at[b]]
            assert (s[b, :, at[b] // block + 1:] == 0).all()
            # One rounding when stored, and one for each time the block grew.
            bound = half_step(w, sc, fmt) * (1 + grown[b, j, :, :at[b], None]) * (1.07 if fmt == "fp8" else 1)
            assert ((got[b, :, :at[b]] - w).abs() <= bound).all()
        # A scale is the largest |x| of its block's rows over M, in fp32, or what an earlier piece needed: never more.
        for b in range(B):
            blocks = -(-at[b] // block)
            padded = torch.zeros(H, blocks * block, D, dtype=torch.float64, device="cuda")
            padded[:, :at[b]] = want[b, :, :at[b]]
            top = padded.view(H, blocks, block, D).abs().amax((2, 3)) / MOST[fmt]
            assert ((s[b, :, :blocks].double() - top).abs() <= top * 2.0 ** -22).all()
    for dt2 in (torch.float32, torch.bfloat16, torch.float16):
        back = q8_restore(cache, None, T, dtype=dt2)
        for b_, c, s in zip(back, (cache.k, cache.v), (cache.k_scales, cache.v_scales)):
            want = (c.float() * s.repeat_interleave(block, 2)[..., None])[:, :, :T].to(dt2)
            assert torch.equal(b_, want.transpose(1, 2))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_store_into_pages_and_strides(cuda, fmt):
    from astc_kv_cuda import Q8Cache, Q8Store, q8_restore
    B, H, D, block = 3, 2, 64, 32
    table = torch.tensor([[4, 1], [0, 5], [2, 7]], dtype=torch.int32, device="cuda")
    cache = Q8Cache.zeros(B, H, 256, D, fmt=fmt, block_tokens=block, page_tokens=128, block_table=table, num_pages=8)
    qkv = torch.randn(B, 250, 3 * H, D + 3, device="cuda").bfloat16()[..., 3:]  # rows that start on odd elements
    start = torch.tensor([0, 6, 3], dtype=torch.int32, device="cuda")
    Q8Store(cache, qkv[:, :, H:2 * H], qkv[:, :, 2 * H:], start).run()
    for j, (got, s) in enumerate(zip(values_of(cache), (cache.k_scales, cache.v_scales))):
        sc = s[table.long()].transpose(1, 2).reshape(B, H, -1).double().repeat_interleave(block, 2)[..., None]
        for b, a in enumerate(start.tolist()):
            want = qkv[b, :, (1 + j) * H:(2 + j) * H].double().transpose(0, 1)
            assert ((got[b, :, a:a + 250] - want).abs() <= half_step(want, sc[b, :, a:a + 250], fmt)).all()
    for unused in (3, 6):
        assert not cache.k.view(torch.int8)[unused].any() and not cache.v_scales[unused].any()
    k, _ = q8_restore(cache, start, 10)
    want = values_of(cache)[0]
    for b, a in enumerate(start.tolist()):
        assert torch.equal(k[b].double(), want[b, :, a:a + 10].transpose(0, 1).float().double())


def test_store_out_of_range(cuda):
    """Rows outside the cache are dropped and reported; the rest is stored."""
    from astc_kv_cuda import Q8Cache, q8_store
    cache = Q8Cache.zeros(3, 1, 64, 16, block_tokens=16)
    cache.status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache._c.status_dev = cache.status.data_ptr()
    x = torch.ones(3, 8, 1, 16, device="cuda")
    q8_store(cache, x, x, torch.tensor([60, -1, 0], dtype=torch.int32, device="cuda"))
    assert int(cache.status) == 1
    k = cache.k  # a block's largest value has code 127
    assert (k[0, 0, 60:] == 127).all() and not k[0, 0, :60].any() and not k[1].any() and (k[2, 0, :8] == 127).all()
    table = torch.tensor([[0], [9]], dtype=torch.int32, device="cuda")
    paged = Q8Cache.zeros(2, 1, 64, 16, block_tokens=16, page_tokens=64, block_table=table, num_pages=2)
    paged.status = torch.zeros(1, dtype=torch.int32, device="cuda")
    paged._c.status_dev = paged.status.data_ptr()
    q8_store(paged, x[:2], x[:2], torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert int(paged.status) == 5 and paged.k[0, 0, :8].all() and not paged.k[1].any()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_store_of_zeros_and_what_is_not_finite(cuda, fmt):
    from astc_kv_cuda import Q8Cache, q8_restore, q8_store
    cache = Q8Cache.zeros(1, 1, 96, 32, fmt=fmt, block_tokens=16)
    x = torch.randn(1, 96, 1, 32, device="cuda")
    x[0, :16] = 0
    x[0, 20, 0, 3] = float("inf")
    x[0, 40, 0, 5] = float("nan")
    x[0, 48:64] = 1e-39
    q8_store(cache, x, x.clone(), torch.zeros(1, dtype=torch.int32, device="cuda"))
    k, v = q8_restore(cache, None, 96)
    assert torch.equal(k.isnan(), v.isnan())
    assert not k[0, :16].any() and k[0, 16:48].isnan().all() and not k[0, 48:64].any()
    assert torch.isfinite(k[0, 64:]).all()
    # A row stored after zeros gets the scale it needs.
    small = torch.full((1, 1, 1, 32), 1e-3, device="cuda")
    cache.k_scales[0, 0, 0] = 0
    q8_store(cache, small, small, torch.full((1,), 5, dtype=torch.int32, device="cuda"))
    k, _ = q8_restore(cache, None, 16)
    assert not k[0, :5].any() and ((k[0, 5] - 1e-3).abs() <= 1e-5).all()


def test_counts_of_zero_write_nothing(cuda):
    from astc_kv_cuda import q8_store
    cache, _, _ = make(2, 1, 64, 32, seed=3)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales)]
    x = torch.randn(2, 4, 1, 32, device="cuda")
    z = torch.zeros(2, dtype=torch.int32, device="cuda")
    q8_store(cache, x, x, z + 7, z)
    q8_store(cache, x[:, :0], x[:, :0], z + 7)
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.v, cache.k_scales, cache.v_scales)))


# ------------------------------------------------------------------ eviction

def plain_choice(w, n, keep, sinks, recent):
    """Kept tokens, ascending: numpy's stable sort on the negated weights, NaN first."""
    if n <= keep:
        return np.arange(n)
    mid = w[sinks:n - recent].astype(np.float64)
    mid = np.where(np.isnan(mid), np.inf, mid) + 0.0
    first = np.isnan(w[sinks:n - recent])
    order = np.lexsort((np.arange(mid.size), -mid, ~first))
    best = np.sort(order[:keep - sinks - recent]) + sinks
    return np.concatenate([np.arange(sinks), best, np.arange(n - recent, n)])


def check_evict(cache, k, v, w, lens, keep, sinks=0, recent=0, *, block=32, page=0, lens_none=False):
    from astc_kv_cuda import Q8Cache, Q8Evict
    B, H, D, fmt = cache.batch, cache.kv_heads, cache.head_dim, cache.fmt
    table, pages = None, 0
    if page:
        per = -(-keep // page)
        pages = B * per + 2
        table = torch.randperm(pages, device="cuda")[:B * per].view(B, per).to(torch.int32)
    dst = Q8Cache.zeros(B, H, keep, D, fmt=fmt, block_tokens=block, page_tokens=page, block_table=table, num_pages=pages)
    for t in (dst.k, dst.v):
        t.view(torch.int8).fill_(55)
    lt = None if lens_none else torch.tensor(lens, dtype=torch.int32, device="cuda")
    kept, out_lens, ow = Q8Evict(cache, dst, w, lt, keep=keep, sinks=sinks, recent=recent).run()
    torch.cuda.synchronize()
    got = values_of(dst)
    wn = w.cpu().numpy()
    for b in range(B):
        n = min(lens[b], keep)
        assert int(out_lens[b]) == n
        for h in range(H):
            want = plain_choice(wn[b, h], lens[b], keep, sinks, recent)
            assert np.array_equal(kept[b, h, :n].cpu().numpy(), want)
            assert (kept[b, h, n:] == -1).all() and not ow[b, h, n:].any()
            at = torch.as_tensor(want, device="cuda").long()
            assert torch.equal(ow[b, h, :n].nan_to_num(7.0), w[b, h, at].nan_to_num(7.0))
            for j, x in enumerate((k, v)):
                rows = x[b, h, at]
                pad = torch.zeros(-(-max(n, 1) // block) * block, D, dtype=torch.float64, device="cuda")
                pad[:n] = rows
                sc = (pad.view(-1, block, D).abs().amax((1, 2)) / MOST[fmt]).repeat_interleave(block)[:n, None]
                assert ((got[j][b, h, :n] - rows).abs() <= half_step(rows, sc, fmt) * (1 + 2.0 ** -10)).all()
                end = min(-(-n // block) * block, got[j].shape[2])
                assert not got[j][b, h, n:end].any()
    return dst, kept


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("T,keep,sinks,recent", [(300, 1, 0, 0), (300, 33, 0, 0), (300, 64, 4, 32), (300, 299, 1, 1), (300, 300, 4, 4),
                                                 (300, 400, 4, 4), (300, 40, 8, 32), (1, 1, 0, 0), (5000, 777, 16, 100), (2049, 1024, 0, 5)])
def test_evict_sizes(cuda, fmt, T, keep, sinks, recent):
    cache, k, v = make(2, 3, T, 64, fmt=fmt, seed=T + keep)
    w = torch.rand(2, 3, cache.max_tokens, device="cuda")
    check_evict(cache, k, v, w, [T, max(T // 2, 1)], keep, sinks, recent)


@pytest.mark.parametrize("D,block,page", [(16, 16, 0), (128, 64, 128), (80, 128, 0), (256, 32, 64)])
def test_evict_layouts(cuda, D, block, page):
    cache, k, v = make(3, 2, 1024, D, block=64, page=256, spare=3, seed=D)
    w = torch.exp(3 * torch.randn(3, 2, 1024, device="cuda"))
    check_evict(cache, k, v, w, [1000, 0, 130], 150, 2, 20, block=block, page=page)
    check_evict(cache, k, v, w, [1024] * 3, 150, 2, 20, block=block, page=page, lens_none=True)


def test_evict_ties_and_odd_weights(cuda):
    """Equal weights go to the lower index; -0 equals 0; infinities, subnormal numbers, negative numbers and NaN have a place."""
    cache, k, v = make(1, 6, 3000, 32, seed=1)
    w = torch.zeros(1, 6, 3008, device="cuda")
    w[0, 1] = torch.randint(0, 4, (3008,), device="cuda").float()
    w[0, 2, ::2] = -0.0
    w[0, 3] = torch.randn(3008, device="cuda") * 1e-42
    w[0, 4] = torch.randn(3008, device="cuda")
    w[0, 4, 7:900:31] = float("inf")
    w[0, 4, 8:900:31] = -float("inf")
    w[0, 5, 100:2000:3] = float("nan")
    for keep, sinks, recent in ((1000, 0, 0), (700, 3, 64), (67, 3, 64), (2999, 0, 1)):
        check_evict(cache, k, v, w, [3000], keep, sinks, recent)


def test_evict_twice_and_attend(cuda):
    """Attention weights that a step adds up decide the eviction; the packed cache then serves the next step."""
    from astc_kv_cuda import Q8Attention, q8_attention
    cache, k, v = make(2, 2, 512, 64, block=32, seed=2)
    w = torch.zeros(2, 2, 512, device="cuda")
    lens = torch.tensor([512, 300], dtype=torch.int32, device="cuda")
    for s in range(3):
        Q8Attention(torch.randn(2, 8, 64, device="cuda").bfloat16(), cache, lens, weights=w).run()
    assert torch.allclose(w.sum(-1), torch.full((2, 2), 12.0, device="cuda"), atol=1e-3)
    dst, kept = check_evict(cache, k, v, w, [512, 300], 100, 4, 16)
    q = torch.randn(2, 1, 8, 64, device="cuda").bfloat16()
    dk, dv = values_of(dst)
    ref, _, _, A, vmax = plain_attention(q, dk, dv, [100, 100], [1, 1])
    out = q8_attention(q, dst, torch.tensor([100, 100], dtype=torch.int32, device="cuda"))
    assert ((out.double() - ref).abs() <= vmax * (2.0 ** -19 * A + 2.0 ** -18)).all()


# -------------------------------------------------------- how they are called

def test_streams_and_graphs(cuda):
    """Calls on another stream than the tensors', and inside a CUDA graph."""
    from astc_kv_cuda import Q8Attention, q8_attention
    cache, k, v = make(2, 2, 700, 64, seed=13)
    q = torch.randn(2, 8, 64, device="cuda").bfloat16()
    lens = torch.tensor([700, 9], dtype=torch.int32, device="cuda")
    want = q8_attention(q, cache, lens)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    outs = [q8_attention(q, cache, lens, stream=side) for _ in range(20)]
    side.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    call = Q8Attention(q, cache, lens)
    call.run(side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call.run()
    lens[0] = 333
    call.out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(call.out, q8_attention(q, cache, lens))


def test_python_refusals(cuda):
    from astc_kv_cuda import Q8Attention, Q8Cache, Q8Evict, Q8Restore, Q8Store
    cache, _, _ = make(2, 2, 64, 64, seed=1)
    q = torch.randn(2, 4, 64, device="cuda")
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    x = torch.randn(2, 3, 2, 64, device="cuda")
    w = torch.zeros(2, 2, 64, device="cuda")
    to = Q8Cache.zeros(2, 2, 32, 64, block_tokens=32)
    z = torch.zeros(2, 2, 64, 64, dtype=torch.int8, device="cuda")
    s = torch.zeros(2, 2, 2, device="cuda")
    refused = [
        lambda: Q8Cache(z, z.clone(), s, s.clone(), block_tokens=24),
        lambda: Q8Cache(z, z.clone(), s, s.clone(), block_tokens=16),
        lambda: Q8Cache(z, z.clone(), s.double(), s.clone(), block_tokens=32),
        lambda: Q8Cache(z, z.cpu(), s, s.clone(), block_tokens=32),
        lambda: Q8Cache(z[..., :40], z[..., :40], s, s, block_tokens=32),
        lambda: Q8Cache(z[..., 8:56], z[..., 8:56], s, s, block_tokens=32),
        lambda: Q8Cache(z, z.clone(), s, s.clone(), block_tokens=32, max_tokens=65),
        lambda: Q8Cache(z, z.clone(), s, s.clone(), block_tokens=32, block_table=i.view(2, 1).long()),
        lambda: Q8Attention(q[0], cache, i),
        lambda: Q8Attention(q[:, :3], cache, i),
        lambda: Q8Attention(q.double(), cache, i),
        lambda: Q8Attention(q.cpu(), cache, i),
        lambda: Q8Attention(q[..., ::2], cache, i),
        lambda: Q8Attention(q, cache, i.long()),
        lambda: Q8Attention(q, cache, i[:1]),
        lambda: Q8Attention(q, cache, i, out_dtype=torch.float64),
        lambda: Q8Attention(q, cache, i, out=torch.empty(2, 4, 32, device="cuda")),
        lambda: Q8Attention(q, cache, i, weights=w[:, :, :32]),
        lambda: Q8Attention(q, cache, i, weights=w.half()),
        lambda: Q8Store(cache, x, x[:, :2], i),
        lambda: Q8Store(cache, x, x.half(), i),
        lambda: Q8Store(cache, x, x, None),
        lambda: Q8Store(cache, x[..., :32], x[..., :32], i),
        lambda: Q8Restore(cache, i, -1),
        lambda: Q8Restore(cache, i, 4, dtype=torch.int32),
        lambda: Q8Evict(cache, to, w, i, keep=33),
        lambda: Q8Evict(cache, to, w, i, keep=0),
        lambda: Q8Evict(cache, to, w, i, keep=8, sinks=4, recent=5),
        lambda: Q8Evict(cache, cache, w, i, keep=8),
        lambda: Q8Evict(cache, to, w[:1], i, keep=8),
        lambda: Q8Evict(cache, Q8Cache(z[:, :, :40].clone(), z[:, :, :40].clone(), s.clone(), s.clone(), block_tokens=32), w, i, keep=8),
    ]
    for n, f in enumerate(refused):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {n} was accepted")
    from astc_kv_cuda import AkvError
    with pytest.raises(AkvError):
        Q8Attention(q, cache, i, split_tokens=10)
