"""The 4-bit KV cache on the GPU against plain implementations in 64 bits.

What is stored. The definition rounds amax * (1/6) to fp32 and fp16, x / scale to
fp32 and e2m1, a rotated key's products and sums to fp32: the plain
implementation does each of these operations in 64 bits and rounds it, and codes
and scales have to be the same bits. A value is code * scale rounded to fp16,
which 64 bits hold before the rounding.

Attention: a score is a sum of D <= 256 products in fp32, in at most 16
accumulating steps that may truncate, so it is off by at most 2^-20 A with A
the largest sum of |scale q k| of a row; that makes every softmax weight off
by a factor of at most 1 +- 2^-19 A, and 2^-18 covers exp2, the running sums
and V's part. An output is a weighted mean of V's rows: the bound is
max |V| (2^-19 A + 2^-18), plus 2^-10 max |V| where the softmax weights are
rounded to fp16 (16-bit outputs), plus half an ulp of the output's type.
"""
import math

import numpy as np
import pytest
import torch

from test_gpu_rotary import places_of, turned

pytestmark = pytest.mark.gpu

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
GROUP = 32


def values(codes, scales):
    """Values, in 64 bits, of codes [n, H, T, D / 2] with scales [n, H, D / 32, T]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    level = torch.tensor(LEVELS + [-x for x in LEVELS], dtype=torch.float64, device=codes.device)
    return (level[c] * scales.double().transpose(-1, -2).repeat_interleave(GROUP, -1)).half().double()


def in_order(x, table):
    """x [pages, H, P, ...] as [B, H, T, ...]."""
    if table is None:
        return x
    x = x[table.long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, *x.shape[4:])


def values_of(cache):
    return [in_order(values(c, s), cache.block_table) for c, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales))]


def make(B, H, T, D, *, page=0, seed=0, spare=0, spread=0.5, size=0.4):
    """A cache of T tokens per sequence filled with random codes and scales, in
    one piece or in shuffled pages; and its K and V [B, H, T, D] in 64 bits."""
    from astc_kv_cuda import Q4Cache
    g = torch.Generator(device="cuda").manual_seed(seed)
    room = -(-T // (page or 16)) * (page or 16)
    per = room // (page or room)
    n = B * per + spare
    table = torch.randperm(n, generator=g, device="cuda")[:B * per].view(B, per).to(torch.int32) if page else None
    sides = []
    for _ in range(2):
        codes = torch.randint(0, 256, (n, H, page or room, D // 2), generator=g, device="cuda", dtype=torch.uint8)
        s = (torch.exp(spread * torch.randn(n, H, D // GROUP, page or room, generator=g, device="cuda")) * size).half()
        sides.append((codes, s))
    cache = Q4Cache(sides[0][0], sides[1][0], sides[0][1], sides[1][1], block_table=table)
    return cache, *values_of(cache)


def plain_attention(q, k, v, lens, q_lens, causal=True, scale=None):
    """out [B, n, Hq, D], lse [B, n, Hq], A and max |V|, in 64 bits."""
    B, n, Hq, D = q.shape
    H, T = k.shape[1], k.shape[2]
    G = Hq // H
    scale = scale or D ** -0.5
    i = torch.arange(n, device=q.device)
    ln = torch.tensor(lens, device=q.device).clamp(0, T).view(B, 1)
    qn = torch.tensor(q_lens, device=q.device).clamp(0, n).view(B, 1)
    ends = torch.where(i < qn, (ln - qn + i + 1).clamp(min=0) if causal else ln.expand(B, n), 0)
    seen = (torch.arange(T, device=q.device) < ends[..., None]).view(B, 1, 1, n, T)
    qq = q.double().view(B, n, H, G, D).permute(0, 2, 3, 1, 4)
    s = (qq.flatten(2, 3) @ k.transpose(-1, -2)).view(B, H, G, n, T) * scale
    a = (qq.abs().flatten(2, 3) @ k.abs().transpose(-1, -2)).view(B, H, G, n, T) * scale
    a = torch.where(seen, a, 0)
    s = torch.where(seen, s, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, (s - torch.where(lse.isinf(), 0, lse)[..., None]).exp(), 0)
    used = torch.where((torch.arange(T, device=q.device) < ln).view(B, 1, T, 1), v, 0)
    out = (p.flatten(2, 3) @ used).view(B, H, G, n, D)
    return (out.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D), lse.permute(0, 3, 1, 2).reshape(B, n, Hq),
            float(a.max()) if a.numel() else 0.0, float(used.abs().max()) if used.numel() else 0.0)


HALF_ULP = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def check_attention(cache, k, v, q, lens, q_lens=None, *, out_dtype=torch.float32, causal=True, scale=0.0, split=0, lens_none=False):
    from astc_kv_cuda import Q4Attention
    B = cache.batch
    rows = q if q.dim() == 4 else q.unsqueeze(1)
    n = rows.shape[1]
    lt = None if lens_none else torch.tensor(lens, dtype=torch.int32, device="cuda")
    qt = torch.tensor(q_lens, dtype=torch.int32, device="cuda") if q_lens is not None else None
    call = Q4Attention(q, cache, lt, q_lens=qt, causal=causal, scale=scale, out_dtype=out_dtype, lse=True, split_tokens=split)
    call.out.fill_(float("nan"))
    call.lse.fill_(float("nan"))
    call.workspace.fill_(255)
    out = call.run().double().view(rows.shape)
    torch.cuda.synchronize()
    ref, lse, A, vmax = plain_attention(rows, k, v, lens, q_lens or [n] * B, causal, scale or None)
    f = 2.0 ** -19 * A + 2.0 ** -18
    tol = vmax * (f + (2.0 ** -10 if out_dtype != torch.float32 else 0.0)) + HALF_ULP[out_dtype] * ref.abs() + 1e-30
    if out_dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a step below its normal numbers
    bad = ~((out - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outputs off, worst {float((out - ref).abs().max()):.3e}, bound {float(tol.max()):.3e}"
    got = call.lse.double()
    assert torch.equal(torch.isinf(got), torch.isinf(lse)) and not torch.isnan(got).any()
    fin = ~torch.isinf(lse)
    assert ((got - lse)[fin].abs() <= f + 2.0 ** -22 * lse[fin].abs()).all()
    return call


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("G,H,D", [(3, 3, 64), (4, 2, 128), (8, 1, 128), (1, 4, 64), (16, 1, 128), (3, 2, 160), (4, 1, 96), (2, 2, 256),
                                   (1, 2, 32), (20, 1, 32), (5, 1, 224), (7, 1, 192)])
def test_one_token_head_layouts(cuda, G, H, D):
    cache, k, v = make(2, H, 300, D, seed=G * D)
    q = torch.randn(2, G * H, D, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [300, 177])
    check_attention(cache, k, v, q, [300, 177], out_dtype=torch.bfloat16)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T", [1, 2, 3, 5, 6, 7, 15, 16, 17, 31, 33, 64, 65, 81, 127, 129, 255, 257, 391, 1025])
def test_one_token_lengths(cuda, T, D):
    cache, k, v = make(3, 2, T + 40, D, seed=T)
    q = torch.randn(3, 6, D, device="cuda").half()
    check_attention(cache, k, v, q, [T, max(T - 1, 0), 0])


@pytest.mark.parametrize("page", [16, 32, 48, 64, 96, 256, 640])
@pytest.mark.parametrize("n", [1, 9, 70])
@pytest.mark.parametrize("D", [128, 256])
def test_pages(cuda, page, n, D):
    cache, k, v = make(4, 2, 1000, D, page=page, spare=5, seed=page + n)
    q = torch.randn(4, n, 8, D, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [1000, n, 255 + n, 513], out_dtype=torch.bfloat16)
    check_attention(cache, k, v, q, [997, 150, 0, 64], [n, 1, n, n - n // 3])


@pytest.mark.parametrize("qd", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("od", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 3, 40])
@pytest.mark.parametrize("D", [64, 128])
def test_types(cuda, qd, od, n, D):
    cache, k, v = make(2, 2, 200, D, seed=n)
    q = torch.randn(2, n, 8, D, device="cuda").to(qd)
    check_attention(cache, k, v, q, [200, 131], out_dtype=od)


@pytest.mark.parametrize("n,T,q_lens,lens", [
    (2, 64, [2, 1], [64, 1]), (5, 130, [5, 3], [130, 3]), (5, 130, [0, 5], [70, 5]), (17, 257, [17, 9], [257, 200]),
    (33, 96, [33, 33], [96, 33]), (64, 64, [64, 1], [64, 64]), (100, 300, [100, 77], [300, 77]), (129, 150, [129, 128], [150, 150]),
    (260, 700, [260, 1], [700, 333]),
    (6, 64, [6, 6], [3, 0]),  # fewer cached tokens than queries: the first queries see nothing
    (90, 200, [90, 90], [50, 0]), (300, 400, [300, 299], [100, 290]),
])
@pytest.mark.parametrize("D,G", [(64, 3), (128, 4)])
@pytest.mark.parametrize("od", [torch.float32, torch.bfloat16])
def test_many_tokens(cuda, n, T, q_lens, lens, D, G, od):
    cache, k, v = make(2, 2, T, D, seed=n + T)
    q = torch.randn(2, n, 2 * G, D, device="cuda").bfloat16()
    check_attention(cache, k, v, q, lens, q_lens, out_dtype=od)


@pytest.mark.parametrize("D,G,n,T", [(256, 4, 9, 40), (256, 8, 33, 300), (224, 2, 64, 129), (160, 1, 200, 517), (256, 1, 33, 33),
                                     (96, 3, 70, 400), (32, 2, 150, 300)])
def test_many_tokens_of_other_heads(cuda, D, G, n, T):
    cache, k, v = make(2, 1, T, D, seed=D + n)
    q = torch.randn(2, n, G, D, device="cuda").half()
    check_attention(cache, k, v, q, [T, max(T // 2, n)], [n, n // 2 + 1], out_dtype=torch.float16)


@pytest.mark.parametrize("n,od", [(1, torch.float32), (3, torch.float32), (20, torch.bfloat16)])
def test_many_sequences(cuda, n, od):
    """More sequences than a CTA has threads, many of them empty."""
    B = 300
    cache, k, v = make(B, 1, 200, 64, seed=n)
    q = torch.randn(B, n, 2, 64, device="cuda").bfloat16()
    r = np.random.default_rng(n)
    lens = [int(x) if x % 3 else 0 for x in r.integers(0, 201, B)]
    q_lens = [int(x) for x in r.integers(0, n + 1, B)]
    check_attention(cache, k, v, q, lens, q_lens, out_dtype=od)
    check_attention(cache, k, v, q, [0] * B, q_lens, out_dtype=od)


@pytest.mark.parametrize("T,lens", [(4096, [4096, 1]), (4000, [63, 0]), (700, [700, 449])])
@pytest.mark.parametrize("G", [1, 4, 8])
def test_one_token_of_few_heads(cuda, T, lens, G):
    cache, k, v = make(2, 2, T, 128, seed=T + G)
    q = torch.randn(2, 2 * G, 128, device="cuda")
    check_attention(cache, k, v, q, lens)
    check_attention(cache, k, v, q.half(), lens, out_dtype=torch.float16)


@pytest.mark.parametrize("D,H,T,lens", [(64, 3, 8192, [8192, 4097]), (128, 1, 8177, [8177, 0]), (256, 1, 8000, [7999, 1]), (128, 2, 8208, [8208, 8193])])
def test_one_token_of_long_sequences(cuda, D, H, T, lens):
    cache, k, v = make(2, H, T, D, seed=T + D, page=48)
    q = torch.randn(2, 4 * H, D, device="cuda")
    check_attention(cache, k, v, q, lens)
    check_attention(cache, k, v, q.bfloat16(), lens, out_dtype=torch.bfloat16)


@pytest.mark.parametrize("D,G,n,T", [(64, 3, 6, 16400), (128, 4, 5, 8190), (128, 1, 31, 8500), (96, 2, 16, 8200), (256, 2, 9, 6000)])
@pytest.mark.parametrize("od", [torch.bfloat16, torch.float16])
def test_few_tokens_of_large_caches(cuda, D, G, n, T, od):
    """Seventeen to thirty-two rows (eighteen above head_dim 128) over long sequences."""
    cache, k, v = make(2, 4, T, D, seed=D + n, page=80)
    q = torch.randn(2, n, 4 * G, D, device="cuda").to(od)
    check_attention(cache, k, v, q, [T, n + 3], [n, n - 2], out_dtype=od)
    check_attention(cache, k, v, q, [T - 130, 1000], out_dtype=od, split=512)


@pytest.mark.parametrize("n", [1, 4, 50])
def test_not_causal_and_scale(cuda, n):
    cache, k, v = make(2, 1, 333, 64, seed=3)
    q = torch.randn(2, n, 5, 64, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [333, 100], causal=False, scale=0.37)
    check_attention(cache, k, v, q, [333, 0], causal=False, out_dtype=torch.float16)


@pytest.mark.parametrize("split", [16, 48, 64, 192, 1024])
@pytest.mark.parametrize("n", [1, 40, 150])
def test_splits_agree(cuda, split, n):
    cache, k, v = make(2, 2, 1000, 128, page=128, seed=9)
    q = torch.randn(2, n, 8, 128, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [1000, 500], split=split)
    check_attention(cache, k, v, q, [1000, 500], split=split, out_dtype=torch.bfloat16)


def test_lens_none_and_long(cuda):
    cache, k, v = make(1, 2, 20000, 64, seed=4)
    q = torch.randn(1, 6, 64, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [cache.max_tokens], lens_none=True)


@pytest.mark.parametrize("n", [1, 30])
def test_scores_and_scales_of_any_size(cuda, n):
    """Peaked softmax (scores of hundreds), V scales over ten decades (subnormal ones too), groups of zeros."""
    from astc_kv_cuda import Q4Cache
    a, _, _ = make(2, 1, 640, 128, seed=5)
    b, _, _ = make(2, 1, 640, 128, seed=5, spread=4.0, size=0.01)
    b.v_scales.clamp_(max=10912)
    for s in (a.k_scales, b.v_scales):
        s[:, :, 1, 96:128] = 0
        s[:, :, :, 333] = 0
    cache = Q4Cache(a.k, b.v, a.k_scales, b.v_scales)
    k, v = values_of(cache)
    q = torch.randn(2, n, 4, 128, device="cuda") * 30
    check_attention(cache, k, v, q, [640, 333])
    q = torch.randn(2, n, 4, 128, device="cuda") * 1e-3
    check_attention(cache, k, v, q.half(), [640, 333], out_dtype=torch.bfloat16)


def test_large_and_tiny_queries(cuda):
    """fp32 queries whose values no 16-bit type holds; the largest keys and values."""
    cache, k, v = make(1, 1, 100, 64, seed=6)
    for f in (1e-20, 1e15):
        q = torch.randn(1, 2, 64, device="cuda") * f
        check_attention(cache, k, v, q, [100], scale=0.1 / f)
    q = torch.randn(1, 40, 2, 64, device="cuda") * 1e30
    check_attention(cache, k, v, q, [100], scale=1e-31)
    cache.k_scales.fill_(10912)
    cache.v_scales.fill_(10912)
    k, v = values_of(cache)
    check_attention(cache, k, v, torch.randn(1, 40, 2, 64, device="cuda").bfloat16(), [100], scale=1e-6, out_dtype=torch.bfloat16)
    check_attention(cache, k, v, torch.randn(1, 2, 64, device="cuda").bfloat16(), [100], scale=1e-6)


@pytest.mark.parametrize("n", [1, 5, 64])
@pytest.mark.parametrize("D,G", [(64, 2), (128, 4), (256, 1)])
def test_what_lies_past_the_length_is_not_read_into_results(cuda, n, D, G):
    cache, k, v = make(2, 2, 256, D, seed=7)
    for lens in ([n + 100, n + 64], [n + 67, n + 1], [n + 130, n + 14]):
        for b in range(2):
            for c, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
                c[b, :, lens[b]:] = 255
                s[b, :, :, lens[b]:] = float("nan") if b else float("inf")
        q = torch.randn(2, n, 2 * G, D, device="cuda").bfloat16()
        check_attention(cache, k, v, q, lens, out_dtype=torch.float32)
        check_attention(cache, k, v, q, lens, out_dtype=torch.bfloat16)
        cache, k, v = make(2, 2, 256, D, seed=8)


@pytest.mark.parametrize("n", [1, 24, 140])
def test_bad_table_entries_read_as_zeros(cuda, n):
    cache, k, v = make(2, 2, 512, 64, page=128, seed=10)
    cache.status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache._c.status_dev = cache.status.data_ptr()
    cache.block_table[0, 1], cache.block_table[1, 2] = 99999, -1
    for x in (k, v):
        x[0, :, 128:256] = 0
        x[1, :, 256:384] = 0
    q = torch.randn(2, n, 4, 64, device="cuda").bfloat16()
    for od in (torch.float32, torch.bfloat16):
        cache.status.zero_()
        check_attention(cache, k, v, q, [512, 300], out_dtype=od)
        assert int(cache.status) == 5


@pytest.mark.parametrize("n", [1, 40])
def test_strided_queries_and_caches(cuda, n):
    """Queries inside a fused projection; codes stored token-major ([B, T, H, D / 2]), scales inside a larger tensor."""
    from astc_kv_cuda import Q4Cache
    base, k, v = make(2, 3, 160, 64, seed=11)
    codes = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in (base.k, base.v)]
    pad = [torch.full((2, 160, 3, 64), 77, dtype=torch.uint8, device="cuda")[..., 16:48].transpose(1, 2) for _ in range(2)]
    for p, c in zip(pad, codes):
        p.copy_(c)
    room = [torch.full((2, 3, 2, 200), float("nan"), dtype=torch.float16, device="cuda")[..., 8:168] for _ in range(2)]
    room[0].copy_(base.k_scales)
    room[1].copy_(base.v_scales)
    for kk, vv, ks, vs in ((codes[0], codes[1], base.k_scales, base.v_scales), (pad[0], pad[1], room[0], room[1])):
        cache = Q4Cache(kk, vv, ks, vs)
        qkv = torch.randn(2, n, 9 + 2 * 3, 64, device="cuda").bfloat16()
        check_attention(cache, k, v, qkv[:, :, :9], [160, 99])
        odd = torch.empty(2, n, 9, 67, dtype=torch.float16, device="cuda")[..., 3:]  # rows on odd elements
        odd.normal_()
        check_attention(cache, k, v, odd, [160, 99], out_dtype=torch.float16)


@pytest.mark.parametrize("n", [1, 64])
def test_runs_repeat_bit_for_bit(cuda, n):
    from astc_kv_cuda import Q4Attention
    cache, _, _ = make(3, 2, 3000, 128, page=256, seed=12)
    q = torch.randn(3, n, 8, 128, device="cuda").bfloat16()
    lens = torch.tensor([3000, 1234, 77], dtype=torch.int32, device="cuda")
    for od in (torch.float32, torch.bfloat16):
        call = Q4Attention(q, cache, lens, out_dtype=od)
        first = call.run().clone()
        for _ in range(5):
            assert torch.equal(call.run(), first)


@pytest.mark.parametrize("D,G,n,od", [(64, 1, 40, torch.bfloat16), (128, 4, 32, torch.bfloat16), (128, 4, 150, torch.bfloat16), (256, 1, 40, torch.bfloat16),
                                      (64, 2, 4, torch.float32), (128, 4, 20, torch.float32), (128, 4, 4, torch.bfloat16), (256, 2, 50, torch.float32),
                                      (224, 2, 90, torch.float16)])
def test_nan_shows_where_it_is_seen(cuda, D, G, n, od):
    """A token with NaN in K's scales among the queries' own: queries that see it are NaN, queries that end before it,
    queries past q_lens and queries that see nothing are as without it."""
    from astc_kv_cuda import Q4Attention
    T = n + 256
    cache, k, v = make(3, 2, T, D, seed=n + D)
    lens, q_lens = [T, T - 5, n // 2], [n, n - 3, n]
    q = torch.randn(3, n, 2 * G, D, device="cuda").bfloat16()
    ref, lse, A, vmax = plain_attention(q, k, v, lens, q_lens)
    at = [lens[b] - 1 - n // 3 for b in range(3)]
    for b in range(3):
        cache.k_scales[b, :, :, at[b]] = float("nan")
        cache.k[b, :, at[b]] = 0
    i32 = dict(dtype=torch.int32, device="cuda")
    call = Q4Attention(q, cache, torch.tensor(lens, **i32), q_lens=torch.tensor(q_lens, **i32), out_dtype=od, lse=True)
    out = call.run().double()
    f = 2.0 ** -19 * A + 2.0 ** -18
    tol = vmax * (f + (0.0 if od == torch.float32 else 2.0 ** -10)) + HALF_ULP[od] * ref.abs() + 2.0 ** -25
    for b in range(3):
        for i in range(n):
            end = lens[b] - q_lens[b] + i + 1 if i < q_lens[b] else 0  # tokens that the query sees
            if end > at[b]:
                assert out[b, i].isnan().all() and call.lse[b, i].isnan().all(), (b, i)
            else:
                assert ((out[b, i] - ref[b, i]).abs() <= tol[b, i]).all(), (b, i)
                assert torch.equal(call.lse[b, i].isinf(), lse[b, i].isinf()) and not call.lse[b, i].isnan().any(), (b, i)


SHAPES = [(64, 1, 40), (128, 4, 32), (128, 2, 100), (64, 3, 90), (128, 4, 150), (256, 1, 40), (224, 2, 90)]


def one_hot(D, G, n, T, size, sign, at, seed):
    """A cache and queries whose scores are `size` times numbers of order one, the one of token `at` far above the
    others. Returns also the score of `at` (scale 1)."""
    cache, _, v = make(1, 2, T, D, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache.k.zero_()
    code = torch.randint(0, 5, cache.k.shape[:3], generator=g, device="cuda", dtype=torch.uint8)  # 0 to 2
    if sign > 0:
        code += 8 * torch.randint(0, 2, code.shape, generator=g, device="cuda", dtype=torch.uint8)
        code[:, :, at] = 7
    else:
        code += 3  # 1.5 to 6
        code[:, :, at] = 1
    cache.k[..., 0] = code
    cache.k_scales.fill_(0.25)
    q = torch.zeros(1, n, 2 * G, D, device="cuda")
    q[..., 0] = sign * size
    return cache, v, q, sign * size * LEVELS[int(code[0, 0, at])] / 4


@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 17, 2.0 ** 22, 2.0 ** 27, 2.0 ** 29, 2.0 ** 33, 2.0 ** 70, 2.0 ** 120])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("D,G,n,T,od", [(D, G, n, n + 333, torch.bfloat16) for D, G, n in SHAPES] + [
    (64, 3, 1, 9000, torch.float32), (128, 4, 1, 5000, torch.float32), (128, 8, 1, 700, torch.float32), (128, 4, 1, 5000, torch.float16),
    (128, 4, 5, 3000, torch.float32), (256, 2, 1, 6000, torch.float32), (128, 4, 20, 2000, torch.float32)])
def test_scores_of_any_magnitude(cuda, D, G, n, T, od, sign, size):
    """One token has all the weight, whatever the size of the scores, also where several CTAs divide a row's tokens; an
    output is its V row, off by the rounding of the weight (to fp16 with 16-bit outputs) and of the output. Tokens that
    are not seen do not count, even where every score is far below 0."""
    from astc_kv_cuda import Q4Attention
    for at in (3, T - n):
        cache, v, q, score = one_hot(D, G, n, T, size, sign, at, seed=n)
        lens = torch.full((1,), T, dtype=torch.int32, device="cuda")
        call = Q4Attention(q if od == torch.float32 else q.bfloat16(), cache, lens, scale=1.0, out_dtype=od, lse=True)
        out = call.run().double().view(1, n, 2, G, D)
        want = v[:, :, at].view(1, 1, 2, 1, D).expand_as(out)
        off = 2.0 ** -18 + (0.0 if od == torch.float32 else 2.0 ** -10) + HALF_ULP[od]
        assert ((out - want).abs() <= off * want.abs() + (2.0 ** -25 if od == torch.float16 else 0.0)).all()
        assert ((call.lse.double() - score).abs() <= 2.0 ** -20 * abs(score) + 2.0 ** -18).all()


# ------------------------------------------------------------------ append

def quantised(x):
    """x [..., D], fp32 numbers in 64 bits -> codes [..., D / 2], scales [..., D / 32]; not for infinities and NaN."""
    x = x.unflatten(-1, (-1, GROUP))
    s = (x.abs().amax(-1) * float(np.float32(1) / np.float32(6))).float().half().double().clamp(max=10912)
    y = torch.where(s[..., None] > 0, x / s.clamp(min=2.0 ** -24)[..., None], 0).float().double()
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    middles = (levels[1:] + levels[:-1]) / 2
    low, high = torch.bucketize(y.abs(), middles), torch.bucketize(y.abs(), middles, right=True)
    c = torch.where(low % 2 == 0, low, high) + 8 * torch.signbit(y).long()  # a middle goes to the even code
    c = c.flatten(-2)
    return (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8), s.half()


def same_codes(got, want):
    """Equal, but for the sign of zeros."""
    for half in (lambda c: c & 15, lambda c: c >> 4):
        a, b = half(got), half(want)
        assert ((a == b) | ((a & 7) + (b & 7) == 0)).all()


def check_append(cache, k, v, start, counts=None, *, rotary=None, places=None, q=None, before=None):
    """Appends, and compares every row of the cache and the rotated queries."""
    from astc_kv_cuda import Q4Append
    i32 = dict(dtype=torch.int32, device="cuda")
    B, n = k.shape[:2]
    T = cache.max_tokens
    old = [(in_order(c, cache.block_table).clone(), in_order(s.transpose(-1, -2), cache.block_table).clone())
           for c, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales))]
    call = Q4Append(cache, k, v, torch.tensor(start, **i32), None if counts is None else torch.tensor(counts, **i32), rotary=rotary,
                    positions=places, q=q)
    if q is not None:
        call.q.fill_(float("nan"))
    got = call.run()
    assert got is (cache if q is None else call.q)
    turn = lambda x: x.double()  # noqa: E731
    if rotary is not None:
        at = places
        if at is None:
            at = (torch.tensor(start, **i32).view(B, 1) + torch.arange(n, **i32)).expand(rotary.axis_count, B, n)
        at = at.view(-1, B, n).clamp(0, rotary.table.shape[0] - 1)
        axes = list(rotary._c.axis)[:rotary.pairs]
        turn = lambda x: turned(x, rotary.table, axes, at, rotary.interleaved)  # noqa: E731
    for (codes, scales), x, c, s in zip(old, (turn(k), v.double()), (cache.k, cache.v), (cache.k_scales, cache.v_scales)):
        wc, ws = quantised(x)
        for b in range(B):
            m = n if counts is None else min(max(counts[b], 0), n)
            m = min(m, T - start[b]) if 0 <= start[b] < T else 0
            if m > 0:
                codes[b, :, start[b]:start[b] + m] = wc[b, :m].transpose(0, 1)
                scales[b, :, start[b]:start[b] + m] = ws[b, :m].transpose(0, 1)
        same_codes(in_order(c, cache.block_table), codes)
        assert torch.equal(in_order(s.transpose(-1, -2), cache.block_table), scales)
    if q is not None:
        want = turn(q)
        if counts is not None:
            want[torch.arange(n, device="cuda") >= torch.tensor(counts, device="cuda").view(B, 1)] = 0
        assert torch.equal(call.q, want.float().to(q.dtype))
    return call


TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("D,R,H,Hq,n", [(128, 128, 8, 32, 33), (64, 64, 3, 9, 7), (128, 64, 2, 16, 5), (256, 128, 1, 8, 19), (96, 96, 4, 12, 21),
                                        (160, 160, 5, 20, 3), (32, 32, 1, 1, 1), (64, 32, 16, 16, 2), (224, 224, 2, 2, 4), (192, 20, 1, 3, 5), (32, 6, 2, 2, 40)])
def test_append_shapes(cuda, D, R, H, Hq, n, dt, interleaved):
    from astc_kv_cuda import Q4Cache, Rotary
    rot = Rotary.make(R, 200, theta=1000.0, interleaved=interleaved)
    cache = Q4Cache.zeros(2, H, 100, D)
    qkv = torch.randn(2, n, Hq + 2 * H, D, device="cuda").to(dt)
    q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + H], qkv[:, :, Hq + H:]
    check_append(cache, k, v, [0, 55], rotary=rot, q=q)
    check_append(cache, k, v, [3, 17], [n, n // 2], rotary=rot, q=q)
    check_append(cache, k, v, [40, 1], [0, n])
    check_append(cache, k, v, [40, 60], rotary=rot, places=places_of(1, 2, n, 200)[0])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("D,R,H,Hq,n", [(128, 128, 8, 32, 64), (64, 64, 3, 9, 71), (128, 64, 2, 16, 133), (256, 128, 1, 8, 66), (256, 256, 2, 2, 65)])
def test_append_many_tokens(cuda, D, R, H, Hq, n, dt):
    from astc_kv_cuda import Q4Cache, Rotary
    rot = Rotary.make(R, 300, theta=1000.0)
    cache = Q4Cache.zeros(2, H, 208, D)
    qkv = torch.randn(2, n, Hq + 2 * H, D, device="cuda").to(dt)
    q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + H], qkv[:, :, Hq + H:]
    check_append(cache, k, v, [0, 55], rotary=rot, q=q)
    check_append(cache, k, v, [3, 17], [n, n // 2], rotary=rot)
    check_append(cache, k, v, [40, 1], [0, n])
    check_append(cache, k, v, [40, 60], rotary=rot, places=places_of(1, 2, n, 300)[0], q=q)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", TYPES)
def test_append_queries_of_thousands_of_tokens(cuda, dt, interleaved):
    from astc_kv_cuda import Q4Cache, Rotary
    n = 4100
    rot = Rotary.make(64, n + 60, sections=(8, 12, 12), interleaved=interleaved)
    cache = Q4Cache.zeros(2, 1, n + 59, 64)
    qkv = torch.randn(2, n, 5, 64, device="cuda").to(dt)
    q, k, v = qkv[:, :, :3], qkv[:, :, 3:4], qkv[:, :, 4:]
    check_append(cache, k, v, [0, 59], [n, n - 37], rotary=rot, q=q)
    check_append(cache, k, v, [59, 1], rotary=rot, places=places_of(3, 2, n, n + 60), q=q)


@pytest.mark.parametrize("sections", [(16, 16), (8, 12, 12)])
@pytest.mark.parametrize("page", [16, 48, 256])
def test_append_axes_into_pages(cuda, sections, page):
    from astc_kv_cuda import Rotary
    cache, _, _ = make(3, 2, 500, 64, page=page, spare=4, seed=page)
    rot = Rotary.make(64, 90, sections=sections)
    k, v = torch.randn(2, 3, 131, 2, 64, device="cuda").half()
    q = torch.randn(3, 131, 6, 64, device="cuda").half()
    check_append(cache, k, v, [0, 15, 369], [131, 99, 131], rotary=rot, places=places_of(len(sections), 3, 131, 90), q=q)


@pytest.mark.parametrize("dt", TYPES)
def test_append_strides(cuda, dt):
    """Rows on odd elements, heads before tokens, a row that a batch shares."""
    from astc_kv_cuda import Q4Cache, Rotary
    rot = Rotary.make(64, 100)
    cache = Q4Cache.zeros(2, 3, 64, 64)
    odd = torch.randn(2, 9, 3, 67, device="cuda").to(dt)[..., 3:]
    heads_first = torch.randn(2, 3, 9, 64, device="cuda").to(dt).transpose(1, 2)
    shared = heads_first[:1].expand(2, 9, 3, 64)
    check_append(cache, odd, heads_first, [0, 8], rotary=rot, q=heads_first)
    check_append(cache, heads_first, odd, [9, 1], rotary=rot, q=odd)
    check_append(cache, shared, shared, [20, 30], rotary=rot, q=shared)


def test_append_values_at_the_borders(cuda):
    """Quotients in the middle between two codes go to the even one: 16-bit values hit them often."""
    from astc_kv_cuda import Q4Cache
    cache = Q4Cache.zeros(1, 4, 4096, 64)
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = torch.randn(2, 1, 4096, 4, 64, generator=g, device="cuda").bfloat16()
    steps = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], device="cuda")
    pick = steps[torch.randint(0, 8, k.shape, generator=g, device="cuda")]
    k = (pick * torch.sign(k.float()) * 2.0 ** torch.randint(-6, 6, (1, 4096, 4, 1), generator=g, device="cuda")).bfloat16()
    k[..., ::32] = k.float().abs().amax(-1, keepdim=True).bfloat16() * 1.0
    check_append(cache, k, v, [0])


def test_append_sizes_from_the_smallest_to_the_largest(cuda):
    """Scales from 2^-24 to their limit; zeros; values beyond the range saturate."""
    from astc_kv_cuda import Q4Cache
    cache = Q4Cache.zeros(1, 1, 256, 64)
    size = 10.0 ** torch.linspace(-9, 37, 200, device="cuda", dtype=torch.float64)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(1, 200, 1, 64, generator=g, device="cuda", dtype=torch.float64) * size.view(1, 200, 1, 1) for _ in range(2))
    k[:, 5], v[:, 9, :, :32] = 0, 0
    check_append(cache, k.float(), v.float(), [0])
    assert cache.k_scales.max() == 10912 and values_of(cache)[0].abs().max() == 65472


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("D,n", [(64, 40), (96, 40), (256, 40), (64, 70), (128, 64), (256, 64)])
def test_append_of_values_that_are_not_finite(cuda, dt, D, n):
    """The token's K gets NaN scales and codes of 0, the groups of V that hold one become 0; other tokens and heads are as ever."""
    from astc_kv_cuda import Q4Cache, q4_append, q4_restore
    cache, clean = Q4Cache.zeros(2, 3, 96, D), Q4Cache.zeros(2, 3, 96, D)
    k, v = torch.randn(2, 2, n, 3, D, device="cuda").to(dt)
    start = torch.zeros(2, dtype=torch.int32, device="cuda")
    q4_append(clean, k, v, start)
    bad = [("k", 0, 7, 1, 5, math.nan), ("v", 0, 8, 2, D - 1, math.inf), ("k", 1, 0, 0, D // 2, -math.inf), ("v", 1, 39, 1, 0, -math.nan),
           ("v", 1, 39, 1, 40, math.inf)]
    for side, b, t, h, d, x in bad:
        (k if side == "k" else v)[b, t, h, d] = x
    q4_append(cache, k, v, start)
    tokens = {(b, h, t) for _, b, t, h, _, _ in bad}
    for b in range(2):
        for h in range(3):
            for t in range(n):
                if (b, h, t) not in tokens:
                    assert torch.equal(cache.k[b, h, t], clean.k[b, h, t]) and torch.equal(cache.k_scales[b, h, :, t], clean.k_scales[b, h, :, t])
                    assert torch.equal(cache.v[b, h, t], clean.v[b, h, t]) and torch.equal(cache.v_scales[b, h, :, t], clean.v_scales[b, h, :, t])
                    continue
                assert not cache.k[b, h, t].any() and cache.k_scales[b, h, :, t].isnan().all()
                for g in range(D // 32):
                    if any((b, t, h, g) == (x[1], x[2], x[3], x[4] // 32) and x[0] == "v" for x in bad):
                        assert not cache.v[b, h, t, 16 * g:16 * g + 16].any() and cache.v_scales[b, h, g, t] == 0
                    else:
                        assert torch.equal(cache.v[b, h, t, 16 * g:16 * g + 16], clean.v[b, h, t, 16 * g:16 * g + 16])
                        assert cache.v_scales[b, h, g, t] == clean.v_scales[b, h, g, t]
    back = q4_restore(cache, None, 40, torch.float32)
    assert back[0][0, 7, 1].isnan().all() and torch.isfinite(back[1]).all()


@pytest.mark.parametrize("paged", [False, True])
def test_append_outside(cuda, paged):
    """Rows past the end and starts outside are dropped and reported; no rows are nowhere outside."""
    from astc_kv_cuda import Q4Cache, Rotary
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    paging = dict(block_table=torch.tensor([[0, 1, 2], [3, 4, 5], [6, 8, 7], [9, 10, 11]], dtype=torch.int32, device="cuda"), page_tokens=32,
                  num_pages=12) if paged else {}
    cache = Q4Cache.zeros(4, 2, 90, 32, status=status, **paging)
    k, v = torch.randn(2, 4, 8, 2, 32, device="cuda").bfloat16()
    q = torch.randn(4, 8, 2, 32, device="cuda").bfloat16()
    rot = Rotary.make(32, 200)
    at = places_of(1, 4, 8, 200)[0]
    check_append(cache, k, v, [3, 80, 0, 31], rotary=rot, places=at, q=q)
    assert int(status) == 0
    check_append(cache, k, v, [-5, 90, 1 << 30, 3], [0, 0, -2, 8], rotary=rot, places=at, q=q)
    assert int(status) == 0
    check_append(cache, k, v, [-5, 85, 1 << 30, 3], rotary=rot, places=at, q=q)
    assert int(status) == 1
    status.zero_()
    check_append(cache, k, v, [90, 1, 1, 3], rotary=rot, places=at, q=q)
    assert int(status) == 1


def test_append_into_bad_pages(cuda):
    from astc_kv_cuda import Q4Cache, q4_append
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    table = torch.tensor([[1, 7]], dtype=torch.int32, device="cuda")
    cache = Q4Cache.zeros(1, 1, 64, 64, page_tokens=32, block_table=table, num_pages=4, status=status)
    k, v = torch.randn(2, 1, 20, 1, 64, device="cuda").half()
    q4_append(cache, k, v, torch.full((1,), 20, dtype=torch.int32, device="cuda"))
    assert int(status) == 5 and cache.k_scales[1, 0, 0, 20:].all() and not cache.k_scales[[0, 2, 3]].any()


def test_append_positions_outside_the_table(cuda):
    """The token's K becomes NaN, its queries too, and V stays."""
    from astc_kv_cuda import Q4Cache, Rotary, q4_append
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = Q4Cache.zeros(1, 2, 64, 64, status=status)
    rot = Rotary.make(64, 10)
    k, v, q = torch.randn(3, 1, 12, 2, 64, device="cuda").half()
    out = q4_append(cache, k, v, torch.zeros(1, dtype=torch.int32, device="cuda"), rotary=rot, q=q)
    assert int(status) == 1
    assert cache.k_scales[0, :, :, :10].isfinite().all() and cache.k_scales[0, :, :, 10:12].isnan().all() and not cache.k[0, :, 10:12].any()
    assert out[:, :10].isfinite().all() and out[:, 10:].isnan().all()
    assert torch.equal(values_of(cache)[1][0, :, :12], values(*[x.transpose(-1, -2) if i else x for i, x in enumerate(quantised(v.double().transpose(1, 2)))])[0])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("page", [0, 48])
@pytest.mark.parametrize("D", [32, 64, 160])
def test_restore(cuda, dt, page, D):
    from astc_kv_cuda import q4_restore
    cache, k, v = make(2, 3, 200, D, page=page, seed=D)
    T = cache.max_tokens
    for start, count in (([0, 0], T), ([7, T - 3], 9), ([-2, T], 5)):
        got = q4_restore(cache, torch.tensor(start, dtype=torch.int32, device="cuda"), count, dt)
        for g, w in zip(got, (k, v)):
            for b in range(2):
                at = torch.arange(start[b], start[b] + count, device="cuda")
                rows = torch.where(((at >= 0) & (at < T))[:, None, None], w[b, :, at.clamp(0, T - 1)].transpose(0, 1), 0)
                assert torch.equal(g[b], rows.float().to(dt))
    assert torch.equal(q4_restore(cache, None, 5, dt)[0], k[:, :, :5].transpose(1, 2).float().to(dt))


# ------------------------------------------------------------ used together

@pytest.mark.parametrize("D,Hq,H,page", [(64, 9, 3, 0), (128, 32, 8, 64), (256, 4, 1, 48)])
def test_prompt_in_chunks_then_decoding(cuda, D, Hq, H, page):
    """Prompts of different lengths come in chunks, then tokens one by one, with the rotation on the way: every output is
    that of attention in 64 bits over the values that the cache holds."""
    from astc_kv_cuda import Q4Attention, Q4Cache, Rotary, q4_append
    i32 = dict(dtype=torch.int32, device="cuda")
    B, T = 3, 320
    table = torch.randperm(B * (-(-T // page)) + 2, device="cuda")[:B * (-(-T // page))].view(B, -1).to(torch.int32) if page else None
    cache = Q4Cache.zeros(B, H, T, D, block_table=table, page_tokens=page, num_pages=B * (-(-T // page)) + 2 if page else 0)
    rot = Rotary.make(D, 400)
    have = [0, 0, 0]
    for news in ([100, 37, 0], [57, 100, 1], [9, 3, 100], [1, 1, 1], [1, 1, 1], [0, 1, 1]):
        n = max(news)
        qkv = torch.randn(B, n, Hq + 2 * H, D, device="cuda").bfloat16()
        start, counts = torch.tensor(have, **i32), torch.tensor(news, **i32)
        q = q4_append(cache, qkv[:, :, Hq:Hq + H], qkv[:, :, Hq + H:], start, counts, rotary=rot, q=qkv[:, :, :Hq])
        have = [a + m for a, m in zip(have, news)]
        k, v = values_of(cache)
        for od in (torch.float32, torch.bfloat16):
            check_attention(cache, k, v, q, have, news, out_dtype=od)


def test_decode_loop_in_a_graph(cuda):
    """Append and attention captured once: each replay takes the lengths and inputs of its step."""
    from astc_kv_cuda import Q4Append, Q4Attention, Q4Cache, Rotary
    B, H, G, D, T = 2, 2, 4, 128, 200
    cache = Q4Cache.zeros(B, H, T, D)
    rot = Rotary.make(D, T)
    qkv = torch.randn(B, 1, H * G + 2 * H, D, device="cuda").half()
    start, lens = torch.zeros(2, B, dtype=torch.int32, device="cuda")
    append = Q4Append(cache, qkv[:, :, H * G:H * G + H], qkv[:, :, H * G + H:], start, rotary=rot, q=qkv[:, :, :H * G])
    attend = Q4Attention(append.q, cache, lens, out_dtype=torch.float16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        append.run()
        attend.run()
    for step in range(150):
        qkv.normal_()
        start.fill_(step)
        lens.fill_(step + 1)
        graph.replay()
    out = attend.out.clone()
    k, v = values_of(cache)
    assert cache.k_scales[:, :, :, :150].all() and not cache.k_scales[:, :, :, 150:].any()
    call = check_attention(cache, k, v, append.q, [150, 150], out_dtype=torch.float16)
    assert torch.equal(call.out, out)


def small_calls():
    """By name, what builds a call, with an input that only the call holds: each call that owns memory."""
    from astc_kv_cuda import Q4Append, Q4Attention, Q4Restore, Rotary, Rotate
    cache, _, _ = make(2, 2, 4096, 64, seed=3)
    rot = Rotary.make(64, 4096)
    q0 = torch.randn(2, 8, 64, device="cuda").bfloat16()
    x0 = torch.randn(2, 50, 12, 64, device="cuda").bfloat16()

    def attention():
        return Q4Attention(q0.clone(), cache)

    def restore():
        return Q4Restore(cache, torch.full((2,), 7, dtype=torch.int32, device="cuda"), 64)

    def append():
        x = x0.clone()
        return Q4Append(cache, x[:, :, 8:10], x[:, :, 10:], torch.full((2,), 9, dtype=torch.int32, device="cuda"), rotary=rot, q=x[:, :, :8])

    def rotation():
        return Rotate(x0.clone(), rot, torch.full((2, 50), 9, dtype=torch.int32, device="cuda"))
    return {"attention": attention, "restore": restore, "append": append, "rotate": rotation}


def results(out):
    return list(out) if isinstance(out, tuple) else [out]


@pytest.mark.parametrize("op", ["attention", "restore", "append", "rotate"])
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
@pytest.mark.parametrize("op", ["attention", "restore", "append", "rotate"])
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


def test_no_sequences_and_no_tokens(cuda):
    from astc_kv_cuda import Q4Append, Q4Attention, Q4Cache, Rotary, q4_restore
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    rot = Rotary.make(64, 10)
    cache = Q4Cache.zeros(0, 2, 128, 64)
    x = torch.randn(0, 3, 2, 64, device="cuda")
    assert Q4Append(cache, x, x, none, rotary=rot, q=x).run().shape == (0, 3, 2, 64)
    assert q4_restore(cache, none, 5)[0].shape == (0, 5, 2, 64)
    assert Q4Attention(torch.randn(0, 7, 8, 64, device="cuda"), cache, none, lse=True).run().shape == (0, 7, 8, 64)
    cache, k, v = make(2, 3, 100, 64, seed=2)
    x = torch.randn(2, 0, 3, 64, device="cuda")
    Q4Append(cache, x, x, torch.zeros(2, dtype=torch.int32, device="cuda")).run()
    assert Q4Attention(torch.randn(2, 0, 6, 64, device="cuda"), cache).run().shape == (2, 0, 6, 64)
    assert torch.equal(values_of(cache)[0], k)


def test_offsets_past_32_bits(cuda):
    """The last sequence of more than 2^32 bytes of codes, and the last pages of such a pool: every call."""
    from astc_kv_cuda import Q4Cache, Rotary, q4_append, q4_restore
    B, H, T, D, n = 66, 8, 131072, 128, 300
    assert B * H * T * D // 2 > 1 << 32
    rot = Rotary.make(D, T)
    for paged in (False, True):
        if paged:
            pages = B * T // 256
            table = torch.tensor([[pages - 1, pages - 5, pages - 2, 3]], dtype=torch.int32, device="cuda")
            cache = Q4Cache(cache.k.view(pages, H, 256, D // 2), cache.v.view(pages, H, 256, D // 2), cache.k_scales.view(pages, H, D // 32, 256),
                            cache.v_scales.view(pages, H, D // 32, 256), block_table=table)
            for t in (cache.k, cache.v, cache.k_scales, cache.v_scales):
                t[-8:].zero_()
                t[3].zero_()
        else:
            cache = Q4Cache.zeros(B, H, T, D)
        b, t = cache.batch, cache.max_tokens
        k, v = torch.randn(2, b, n, H, D, device="cuda").bfloat16()
        q = torch.randn(b, n, 2 * H, D, device="cuda").bfloat16()
        q = q4_append(cache, k, v, torch.full((b,), t - n, dtype=torch.int32, device="cuda"), rotary=rot, q=q)
        back = q4_restore(cache, torch.full((b,), t - n, dtype=torch.int32, device="cuda"), n, torch.float32)
        at = torch.arange(t - n, t, device="cuda", dtype=torch.int32).expand(1, b, n)
        kv = []
        for got, x in zip(back, (turned(k, rot.table, [0] * (D // 2), at, False), v.double())):
            c, s = quantised(x[-1:].transpose(1, 2))
            want = values(c, s.transpose(-1, -2))
            assert torch.equal(got[-1:].double(), want.transpose(1, 2))
            kv.append(want[0])
        for m, od in ((1, torch.float32), (n, torch.bfloat16), (20, torch.float32)):
            check_last(cache, kv[0], kv[1], q[:, n - m:], m, od)


def check_last(cache, k, v, q, m, od):
    """The last sequence's attention; of its tokens the last n are k, v [H, n, D], all others zeros."""
    from astc_kv_cuda import Q4Attention
    H, n, D = k.shape
    T, G = cache.max_tokens, q.shape[2] // H
    out = Q4Attention(q.contiguous(), cache, out_dtype=od).run()[-1].double()
    qq = q[-1].double().view(m, H, G, D).permute(1, 2, 0, 3)
    s = torch.einsum("hgmd,htd->hgmt", qq, k) * D ** -0.5
    A = float(torch.einsum("hgmd,htd->hgmt", qq.abs(), k.abs()).max()) * D ** -0.5
    hidden = torch.arange(n, device="cuda") > torch.arange(n - m, n, device="cuda").view(m, 1)
    e = s.masked_fill(hidden, -math.inf).exp()
    p = e / (e.sum(-1, keepdim=True) + (T - n))  # every other token has score 0 and value 0
    ref = torch.einsum("hgmt,htd->mhgd", p, v).reshape(m, H * G, D)
    tol = float(v.abs().max()) * (2.0 ** -19 * A + 2.0 ** -18 + (0.0 if od == torch.float32 else 2.0 ** -10)) + HALF_ULP[od] * ref.abs()
    assert ((out - ref).abs() <= tol).all()


def test_long_sums(cuda):
    """Equal weights over a long sequence: the sum of V's rows must not shrink as the tensor cores truncate. Bounds: fp32 outputs
    2^-18 of max |V|; 16-bit ones 6e-9 a token of a split more (bf16 64 splits of 2048 tokens and more), and their rounding."""
    from astc_kv_cuda import Q4Attention, Q4Cache
    T, D = 131072, 128
    cache = Q4Cache.zeros(1, 1, T, D)
    cache.v.fill_(0x77)
    cache.v_scales.fill_(0.3)
    want = float(torch.tensor(0.3).half() * 6)
    for n, od, off in ((1, torch.float32, 2.0 ** -18), (3, torch.float32, 2.0 ** -18), (1, torch.float16, 2.0 ** -10), (300, torch.bfloat16, 2.0 ** -8 + 1e-3)):
        q = torch.randn(1, n, 4, D, device="cuda").bfloat16()
        out = Q4Attention(q, cache, out_dtype=od).run().double()
        assert ((out - want).abs() <= off * want).all(), (n, float((out - want).abs().max()))


def test_refusals(cuda):
    from astc_kv_cuda import Q4Append, Q4Attention, Q4Cache, Q4Restore, Rotary
    from astc_kv_cuda import AkvError
    cache, _, _ = make(2, 2, 96, 64, page=32)
    c, s, table = cache.k, cache.k_scales, cache.block_table
    for args, kw in [((c, c, s, s), dict(block_table=table.long())), ((c, c, s, s), dict(block_table=table[0])), ((c[:, :, :24], c[:, :, :24], s, s), {}),
                     ((c, c[:1], s, s), {}), ((c, c, s[..., :16], s), {}), ((c, c, s.float(), s), {}), ((c, c, s.transpose(2, 3), s), {}),
                     ((c, c, s, s), dict(max_tokens=1 << 20)), ((c, c, s, s), dict(max_tokens=-1)), ((c, c, s, s), dict(status=table.float())),
                     ((c, c, s, s.cpu()), {}), ((c[..., :24], c[..., :24], s, s), {}), ((c.view(torch.int8), c, s, s), {})]:
        with pytest.raises(ValueError):
            Q4Cache(*args, **kw)
    q = torch.randn(2, 4, 64, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    for a, kw in [((q, cache, lens.long()), {}), ((q, cache, lens[:1]), {}), ((q[:, :3], cache), {}), ((q[..., :32], cache), {}), ((q.double(), cache), {}),
                  ((q[0], cache), {}), ((q, cache), dict(out_dtype=torch.int32)), ((q, cache), dict(out=torch.empty(2, 4, 32, device="cuda"))),
                  ((q, cache), dict(q_lens=lens.float())), ((q.cpu(), cache), {})]:
        with pytest.raises(ValueError):
            Q4Attention(*a, **kw)
    for kw in (dict(split_tokens=24), dict(scale=-1.0)):
        with pytest.raises(AkvError):
            Q4Attention(q, cache, **kw)
    k = torch.randn(2, 5, 2, 64, device="cuda")
    rot = Rotary.make(64, 10)
    at = torch.zeros(2, 5, dtype=torch.int32, device="cuda")
    for a, kw in [((k, k, None), {}), ((k, k.half(), lens), {}), ((k[:, :, :1], k, lens), {}), ((k, k, lens), dict(q=k)), ((k, k, lens), dict(positions=at)),
                  ((k, k, lens), dict(rotary=rot, positions=at[:, :4])), ((k, k, lens), dict(rotary=rot, q=k.half())), ((k, k, lens), dict(rotary=rot, q=k[:, :4])),
                  ((k, k, lens, lens.long()), {}), ((k, k, lens), dict(rotary=Rotary.make(128, 10))), ((k[0], k, lens), {}), ((k, k, lens.cpu()), {})]:
        with pytest.raises(ValueError):
            Q4Append(cache, *a, **kw)
    for a in ((None, -1), (lens.long(), 4), (None, 4, torch.int32)):
        with pytest.raises(ValueError):
            Q4Restore(cache, *a)
