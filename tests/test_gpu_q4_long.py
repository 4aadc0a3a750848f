"""Long sums in the 4-bit cache's attention.

Every token has the same score, so an output is the mean of V's values over all
tokens, which 64 bits hold; V's values are positive and the means lie anywhere between two
numbers of the output's type, so that what a sum loses shows in the mean of the
relative errors. Tensor cores truncate as they add: about 2^-27.3 of a sum is lost with
every token that they add up, here taken as 2^-27. The rounding of an output is off by 2^-11 (fp16),
2^-8 (bf16) at most and at random, evenly spread in between: divided by
the root of 3 one standard deviation, of the mean of 256 values a sixteenth of
that; four of those are 2^-13.8 and 2^-10.8 times the root of 1/3, below 2^-13 and 2^-10 by far.
All sequences read one page.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

P = 1024
NOISE = {torch.float16: 4 * 2.0 ** -11 / 3 ** 0.5 / 16, torch.bfloat16: 4 * 2.0 ** -8 / 3 ** 0.5 / 16}


def one_page(B, H, T, D):
    """A cache of B sequences of T tokens that are all the same page, keys of 0, and V's mean [H, D]."""
    from astc_kv_cuda import Q4Cache
    from test_gpu_q4 import values
    g = torch.Generator(device="cuda").manual_seed(T + D)
    k = torch.zeros(1, H, P, D // 2, dtype=torch.uint8, device="cuda")
    ks = torch.ones(1, H, D // 32, P, dtype=torch.float16, device="cuda")
    c = torch.randint(1, 8, (2, 1, H, P, D // 2), generator=g, device="cuda", dtype=torch.uint8)
    v = c[0] | c[1] << 4
    vs = (1 + torch.rand(1, H, D // 32, P, generator=g, device="cuda")).half()
    table = torch.zeros(B, T // P, dtype=torch.int32, device="cuda")
    return Q4Cache(k, v, ks, vs, block_table=table), values(v, vs)[0].mean(1)


def lost(B, H, T, D, n, od, split):
    """The mean relative error of each row and of all of its values."""
    from astc_kv_cuda import Q4Attention
    assert H * D == 256
    cache, mean = one_page(B, H, T, D)
    q = torch.randn(B, n, H, D, device="cuda").half()
    out = Q4Attention(q, cache, out_dtype=od, causal=False, split_tokens=split).run().double()
    return (out / mean - 1).mean((-2, -1))


@pytest.mark.parametrize("D,n,od,T,split", [
    # Row tiles for every SM, so that nothing but length asks for splits; splits as long as the cache.
    (64, 100, torch.float16, 1 << 17, 0), (64, 100, torch.float16, 1 << 17, 1 << 17), (128, 300, torch.float16, 1 << 17, 1 << 17),
    (256, 100, torch.float16, 1 << 17, 1 << 17),
    (64, 100, torch.bfloat16, 1 << 20, 0), (64, 300, torch.bfloat16, 1 << 20, 0), (128, 100, torch.bfloat16, 1 << 20, 1 << 20),
    (256, 40, torch.bfloat16, 1 << 20, 0)])
def test_many_rows_of_16_bits(cuda, D, n, od, T, split):
    """Sums of 16384 tokens at most with fp16 outputs, of 131072 with bf16 ones."""
    most = 16384 if od == torch.float16 else 131072
    off = lost(148 if n <= 128 else 74, 256 // D, T, D, n, od, split)
    assert (off.abs() <= most * 2.0 ** -27 + NOISE[od]).all(), float(off.abs().max())


@pytest.mark.parametrize("od", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,n", [(64, 1), (64, 16), (128, 1), (128, 9), (256, 1)])
def test_few_rows_of_16_bits(cuda, D, n, od):
    """As many sequences as there are CTAs, so that each goes through all tokens of one, four warps each."""
    most = 16384 if od == torch.float16 else 131072
    off = lost(148 * 4 * D // 256 if n == 1 and D < 256 else 296 * D // 256, 256 // D, (1 << 20 if od == torch.float16 else 1 << 21), D, n, od, 0)
    assert (off.abs() <= most * 2.0 ** -27 + NOISE[od]).all(), float(off.abs().max())


def test_splits_stay_what_was_asked_for_where_sums_are_short(cuda):
    """The longest sum bounds splits from above alone: the workspace of shorter ones is that of a library's choice of them."""
    from astc_kv_cuda import Q4Attention
    cache, _ = one_page(1, 4, 1 << 18, 64)
    q = torch.randn(1, 300, 4, 64, device="cuda").half()
    size = {s: Q4Attention(q, cache, out_dtype=torch.bfloat16, split_tokens=s).workspace.numel() for s in (32768, 65536, 131072, 262144)}
    assert size[32768] > size[65536] > size[131072] == size[262144]


def two_pages(B, T, D, H, kinds, weight):
    """Order of the pages [T / P], 0 and 1, and q [B, 1, H, D], alike in all channels: keys of the first page are 0, of the second 1 in
    every channel, which then weighs exp(q D / sqrt(D)) times as much, 150 to 3000."""
    n = T // P
    order = torch.zeros(n, dtype=torch.long, device="cuda")
    order[kinds[0] * n // 16:kinds[1] * n // 16] = 1
    a = torch.arange(40, 40 + B * H, device="cuda").remainder(24).add(40).view(B, 1, H, 1) / 64 * weight
    return order, a.expand(B, 1, H, D).half().contiguous()


def weighted(order, log_weight, means):
    """Softmax means [B, 1, H, D] of two pages' means [2, H, D]."""
    n1 = int(order.sum())
    w = torch.exp(log_weight)[..., None] * n1
    return (means[0] * (len(order) - n1) + means[1] * w) / (len(order) - n1 + w)


@pytest.mark.parametrize("od,T", [(torch.float16, 1 << 17), (torch.bfloat16, 1 << 20)])
@pytest.mark.parametrize("kinds", [(15, 16), (9, 10), (0, 1), (3, 14)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_largest_scores_anywhere_in_long_sums(cuda, D, kinds, od, T):
    """Sums are put by under one base and joined under another. A weight is one of two numbers, rounded to fp16 (2^-11); sums lose 2^-27 a
    token, and an output is rounded."""
    from astc_kv_cuda import Q4Attention, Q4Cache
    from test_gpu_q4 import HALF_ULP, values
    H = 256 // D
    B = 148 * (4 if D < 256 else 2) // H
    g = torch.Generator(device="cuda").manual_seed(D)
    c = torch.randint(1, 8, (2, 2, H, P, D // 2), generator=g, device="cuda", dtype=torch.uint8)
    v, vs = c[0] | c[1] << 4, (1 + torch.rand(2, H, D // 32, P, generator=g, device="cuda")).half()
    k = torch.zeros(2, H, P, D // 2, dtype=torch.uint8, device="cuda")
    k[1] = 0x22
    order, q = two_pages(B, T, D, H, kinds, (64 / D) ** 0.5)
    cache = Q4Cache(k, v, torch.ones_like(vs), vs, block_table=order.to(torch.int32).expand(B, -1).contiguous())
    log_weight = q[..., 0].double() * D ** 0.5
    out = Q4Attention(q, cache, out_dtype=od, causal=False).run().double()
    want = weighted(order, log_weight, values(v, vs).mean(2))
    most = 16384 if od == torch.float16 else 131072
    assert ((out / want - 1).abs() <= 2.0 ** -11 + 2.0 ** -18 + most * 2.0 ** -27 + HALF_ULP[od]).all(), float((out / want - 1).abs().max())
