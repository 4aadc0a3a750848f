"""A layer's life with an 8-bit KV cache: a prompt comes in chunks, the tokens
that received little attention are evicted, decoding goes on in the smaller
cache. Every result is compared with attention in fp32 over the exact K and V
of the tokens that the cache holds.

    python examples/q8_serving.py [--format int8|fp8] [--prompt 4096] [--keep 1024] [--steps 32]

Shapes are Llama-3-8B's (32 query heads, 8 KV heads, head_dim 128); values are
random.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "astc-kv_b200"))
from astc_kv_cuda import Q8Attention, Q8Cache, Q8Evict, q8_attention, q8_store  # noqa: E402

B, HQ, H, D, PAGE = 2, 32, 8, 128, 256


def exact(q, k, v, seen):
    """fp32 attention of q [B, n, HQ, D] over k, v [B, H, T, D]; query i sees seen[i] tokens."""
    n, t = q.shape[1], k.shape[2]
    qq = q.float().view(B, n, H, HQ // H, D)
    s = torch.einsum("bnhgd,bhtd->bhgnt", qq, k) * D ** -0.5
    s = s.masked_fill(torch.arange(t, device=q.device) >= seen.view(n, 1), float("-inf"))
    return torch.einsum("bhgnt,bhtd->bnhgd", s.softmax(-1), v).reshape(B, n, HQ, D)


def report(what, got, want):
    rel = ((got.float() - want).norm() / want.norm()).item()
    print(f"{what:44s} off fp32 attention by {rel:.2e}")
    return rel


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--format", default="int8", choices=("int8", "fp8"))
    ap.add_argument("--prompt", type=int, default=4096)
    ap.add_argument("--keep", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args()
    torch.manual_seed(0)
    i32 = dict(dtype=torch.int32, device="cuda")

    # A paged cache for the prompt: every sequence's pages anywhere in the pool.
    per = -(-a.prompt // PAGE)
    table = torch.randperm(B * per, device="cuda").view(B, per).to(torch.int32)
    cache = Q8Cache.zeros(B, H, a.prompt, D, fmt=a.format, block_tokens=64, page_tokens=PAGE, block_table=table, num_pages=B * per)
    weights = torch.zeros(B, H, a.prompt, device="cuda")
    start, lens = torch.zeros(B, **i32), torch.zeros(B, **i32)
    k = torch.zeros(B, H, a.prompt, D, device="cuda")
    v = torch.zeros_like(k)
    worst = 0.0
    for at in range(0, a.prompt, 1000):
        n = min(1000, a.prompt - at)
        qkv = torch.randn(B, n, HQ + 2 * H, D, device="cuda").bfloat16()  # a fused projection, read in place
        q, kk, vv = qkv[:, :, :HQ], qkv[:, :, HQ:HQ + H], qkv[:, :, HQ + H:]
        start.fill_(at)
        lens.fill_(at + n)
        q8_store(cache, kk, vv, start)
        out = q8_attention(q, cache, lens, out_dtype=torch.bfloat16, weights=weights)
        k[:, :, at:at + n], v[:, :, at:at + n] = kk.transpose(1, 2).float(), vv.transpose(1, 2).float()
        seen = torch.arange(at + 1, at + n + 1, device="cuda")
        worst = max(worst, report(f"prompt tokens {at} to {at + n}", out, exact(q, k, v, seen)))

    # The tokens that the prompt attended to least make room.
    small = Q8Cache.zeros(B, H, a.keep + a.steps, D, fmt=a.format, block_tokens=64)
    kept, lens, left = Q8Evict(cache, small, weights, lens, keep=a.keep, sinks=4, recent=64).run()
    print(f"{cache.nbytes / 2**20:.1f} MiB of cache are now {small.nbytes / 2**20:.1f} MiB; {left.sum() / weights.sum():.1%} of the weight stays")
    kept_rows = kept.clamp(min=0).long()[..., None].expand(-1, -1, -1, D)
    k, v = (torch.cat([x.gather(2, kept_rows), x.new_zeros(B, H, a.steps, D)], 2) for x in (k, v))

    # Decoding: prepared once, run every step; lengths advance in place.
    q = torch.zeros(B, HQ, D, dtype=torch.bfloat16, device="cuda")
    call = Q8Attention(q, small, lens, weights=left)
    for step in range(a.steps):
        n = a.keep + step
        qkv = torch.randn(B, 1, HQ + 2 * H, D, device="cuda").bfloat16()
        q.copy_(qkv[:, 0, :HQ])
        q8_store(small, qkv[:, :, HQ:HQ + H], qkv[:, :, HQ + H:], lens)
        lens += 1
        out = call.run()
        k[:, :, n], v[:, :, n] = qkv[:, 0, HQ:HQ + H].float(), qkv[:, 0, HQ + H:].float()
        if step in (0, a.steps - 1):
            seen = torch.full((1,), n + 1, device="cuda")
            worst = max(worst, report(f"decode step {step}, {n + 1} tokens", out[:, None], exact(q[:, None], k, v, seen)))
    # Rounding of K and V to 8 bits: half a step of a block's largest value for
    # each of them, a few per cent of what random values average to.
    if not worst < 0.08:
        raise SystemExit(f"the outputs are {worst:.2e} off")


if __name__ == "__main__":
    main()
