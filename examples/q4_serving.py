"""A layer's life with a 4-bit KV cache: a prompt comes in chunks, then tokens
one by one in a CUDA graph. Keys and queries are rotated by their positions on
the way. Every result is compared with attention in fp32, over the values that
the cache holds and over the exact keys and values.

    python examples/q4_serving.py [--prompt 4096] [--steps 32] [--page 64]

Shapes are 32 query heads, 8 KV heads and head_dim 128; values are random.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "astc-kv_b200"))
from astc_kv_cuda import Q4Append, Q4Attention, Q4Cache, Rotary, q4_append, q4_attention, q4_restore, rotate  # noqa: E402

B, HQ, H, D = 2, 32, 8, 128


def exact(q, k, v, seen):
    """fp32 attention of q [B, n, HQ, D] over k, v [B, T, H, D]; query i sees seen[i] tokens."""
    n, t = q.shape[1], k.shape[1]
    qq = q.float().view(B, n, H, HQ // H, D)
    s = torch.einsum("bnhgd,bthd->bhgnt", qq, k.float()) * D ** -0.5
    s = s.masked_fill(torch.arange(t, device=q.device) >= seen.view(n, 1), float("-inf"))
    return torch.einsum("bhgnt,bthd->bnhgd", s.softmax(-1), v.float()).reshape(B, n, HQ, D)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--prompt", type=int, default=4096)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--page", type=int, default=64)
    a = ap.parse_args()
    torch.manual_seed(0)
    i32 = dict(dtype=torch.int32, device="cuda")

    # Every sequence's pages anywhere in the pool.
    room = a.prompt + a.steps
    per = -(-room // a.page)
    table = torch.randperm(B * per, device="cuda").view(B, per).to(torch.int32)
    status = torch.zeros(1, **i32)
    cache = Q4Cache.zeros(B, H, room, D, page_tokens=a.page, block_table=table, num_pages=B * per, status=status)
    rotary = Rotary.make(D, room, theta=500000.0)
    start, lens = torch.zeros(B, **i32), torch.zeros(B, **i32)
    keys, values = (torch.zeros(B, room, H, D, device="cuda") for _ in range(2))
    worst = 0.0

    def report(what, out, q, end, n):
        nonlocal worst
        seen = torch.arange(end - n + 1, end + 1, device="cuda")
        held = [x[:, :end] for x in q4_restore(cache, None, end)]
        want = exact(q, *held, seen)
        rel = ((out.float() - want).norm() / want.norm()).item()
        full = exact(q, keys[:, :end], values[:, :end], seen)
        print(f"{what:32s} off fp32 attention by {rel:.1e}, off that of the exact keys and values by {((out.float() - full).norm() / full.norm()).item():.1e}")
        worst = max(worst, rel)

    def keep(k, v, at, n):
        places = torch.arange(at, at + n, **i32).expand(B, n).contiguous()
        keys[:, at:at + n], values[:, at:at + n] = rotate(k.float(), rotary, places), v.float()

    for at in range(0, a.prompt, 1000):
        n = min(1000, a.prompt - at)
        qkv = torch.randn(B, n, HQ + 2 * H, D, device="cuda").bfloat16()  # a fused projection, read in place
        k, v = qkv[:, :, HQ:HQ + H], qkv[:, :, HQ + H:]
        start.fill_(at)
        lens.fill_(at + n)
        q = q4_append(cache, k, v, start, rotary=rotary, q=qkv[:, :, :HQ])
        out = q4_attention(q, cache, lens, out_dtype=torch.bfloat16)
        keep(k, v, at, n)
        report(f"prompt tokens {at} to {at + n}", out, q, at + n, n)

    # Decoding: captured once, replayed every step; lengths advance in the graph.
    qkv = torch.zeros(B, 1, HQ + 2 * H, D, dtype=torch.bfloat16, device="cuda")
    start.fill_(a.prompt)
    lens.fill_(a.prompt)
    append = Q4Append(cache, qkv[:, :, HQ:HQ + H], qkv[:, :, HQ + H:], start, rotary=rotary, q=qkv[:, :, :HQ])
    attend = Q4Attention(append.q, cache, lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens += 1
        append.run()
        attend.run()
        start += 1
    for step in range(a.steps):
        qkv.normal_()
        graph.replay()
        keep(qkv[:, :, HQ:HQ + H], qkv[:, :, HQ + H:], a.prompt + step, 1)
        if step in (0, a.steps - 1):
            report(f"decode step {step}", attend.out, append.q, a.prompt + step + 1, 1)
    if status.item():
        raise SystemExit(f"a kernel reported {status.item()}")
    # Softmax weights and outputs of the prompt are rounded to 16 bits, 2^-9 of
    # themselves at most; the cache's own rounding is in both sides.
    if not worst < 2.0 ** -8:
        raise SystemExit(f"the outputs are {worst:.2e} off")


if __name__ == "__main__":
    main()
