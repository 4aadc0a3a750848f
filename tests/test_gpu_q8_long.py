"""Long sums of 16-bit outputs in the 8-bit cache's attention: as test_gpu_q4_long.py, which has the bounds,
with scores that differ."""
import pytest
import torch

from test_gpu_q4_long import NOISE, P

pytestmark = pytest.mark.gpu


def lost(B, H, T, D, n, od, split, fmt):
    """The mean relative error of each row's values. Every sequence is the same page over and over, so an output is its mean over one
    page. (Weights have to differ: sums of whole numbers lose nothing for long.)"""
    from astc_kv_cuda import Q8Attention, Q8Cache
    assert H * D == 256
    g = torch.Generator(device="cuda").manual_seed(T + D)
    dt = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    k = torch.randint(-100, 101, (1, H, P, D), generator=g, device="cuda").float().to(dt)
    v = torch.randint(32, 120, (1, H, P, D), generator=g, device="cuda").float().to(dt)
    scales = 1 + torch.rand(1, H, 1, generator=g, device="cuda").expand(1, H, P // 64).contiguous()
    cache = Q8Cache(k, v, torch.full_like(scales, 0.01), scales, block_table=torch.zeros(B, T // P, dtype=torch.int32, device="cuda"))
    q = torch.randn(1, n, H, D, generator=g, device="cuda").half()
    out = Q8Attention(q.expand(B, n, H, D), cache, out_dtype=od, causal=False, split_tokens=split).run().double()
    s = torch.einsum("nhd,htd->nht", q[0].double(), k[0].double() * float(torch.tensor(0.01))) * D ** -0.5
    mean = torch.einsum("nht,htd->nhd", s.softmax(-1), v[0].double()) * scales[0, :, :1].double()
    return (out / mean - 1).mean((-2, -1))


# Weights are rounded to fp16, off by 2^-11 at most and evenly spread. The products of 1024 tokens count as 256 equal ones at
# least: one standard deviation is 2^-11 over the roots of 3 and 256, here four of them.
WEIGHTS = 4 * 2.0 ** -11 / 3 ** 0.5 / 16


@pytest.mark.parametrize("D,n,od,T,split,fmt", [
    (64, 100, torch.float16, 1 << 17, 0, "int8"), (64, 100, torch.float16, 1 << 17, 1 << 17, "fp8"), (128, 300, torch.float16, 1 << 17, 1 << 17, "int8"),
    (256, 100, torch.float16, 1 << 17, 1 << 17, "int8"),
    (64, 100, torch.bfloat16, 1 << 20, 0, "int8"), (64, 300, torch.bfloat16, 1 << 20, 0, "fp8"), (128, 100, torch.bfloat16, 1 << 20, 1 << 20, "int8"),
    (256, 40, torch.bfloat16, 1 << 20, 0, "int8")])
def test_many_rows_of_16_bits(cuda, D, n, od, T, split, fmt):
    """Sums of 16384 tokens at most with fp16 outputs, of 131072 with bf16 ones."""
    most = 16384 if od == torch.float16 else 131072
    off = lost(148 if n <= 128 else 74, 256 // D, T, D, n, od, split, fmt)
    assert (off.abs() <= most * 2.0 ** -27 + NOISE[od] + WEIGHTS).all(), float(off.abs().max())


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("od", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,n", [(64, 1), (64, 16), (128, 1), (128, 9), (256, 1)])
def test_few_rows_of_16_bits(cuda, D, n, od, fmt):
    """As many sequences as there are CTAs, so that each goes through all tokens of one, four warps each."""
    most = 16384 if od == torch.float16 else 131072
    off = lost(148 * 4 * D // 256 if n == 1 and D < 256 else 296 * D // 256, 256 // D, (1 << 20 if od == torch.float16 else 1 << 21), D, n, od, 0, fmt)
    assert (off.abs() <= most * 2.0 ** -27 + NOISE[od] + WEIGHTS).all(), float(off.abs().max())


@pytest.mark.parametrize("od,T", [(torch.float16, 1 << 17), (torch.bfloat16, 1 << 20)])
@pytest.mark.parametrize("kinds", [(15, 16), (9, 10), (0, 1), (3, 14)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_largest_scores_anywhere_in_long_sums(cuda, D, kinds, od, T):
    """As with 4 bits; the power of two that a weight is rounded with holds V's scale, here one number."""
    from astc_kv_cuda import Q8Attention, Q8Cache
    from test_gpu_q4 import HALF_ULP
    from test_gpu_q4_long import two_pages, weighted
    H = 256 // D
    B = 148 * (4 if D < 256 else 2) // H
    g = torch.Generator(device="cuda").manual_seed(D)
    v = torch.randint(32, 120, (2, H, P, D), generator=g, device="cuda").to(torch.int8)
    k = torch.zeros_like(v)
    k[1] = 64
    scales = torch.full((2, H, P // 64), 1 / 64, device="cuda")
    order, q = two_pages(B, T, D, H, kinds, (64 / D) ** 0.5)
    cache = Q8Cache(k, v, scales, torch.ones_like(scales), block_table=order.to(torch.int32).expand(B, -1).contiguous())
    out = Q8Attention(q, cache, out_dtype=od, causal=False).run().double()
    want = weighted(order, q[..., 0].double() * D ** 0.5, v.double().mean(2))
    most = 16384 if od == torch.float16 else 131072
    assert ((out / want - 1).abs() <= 2.0 ** -11 + 2.0 ** -18 + most * 2.0 ** -27 + HALF_ULP[od]).all(), float((out / want - 1).abs().max())
