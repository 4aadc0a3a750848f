"""The 4-bit cache's calls in uses that meet each other: queries that are not
finite next to others, pages that sequences share, calls at the same time on
several streams, outputs on top of inputs, a rotation's backward pass in a CUDA
graph."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from test_gpu_q4 import HALF_ULP, check_attention, make, plain_attention, values_of

pytestmark = pytest.mark.gpu
i32 = dict(dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("D,H,n,od", [(128, 2, 1, torch.float32), (64, 3, 4, torch.bfloat16), (128, 2, 9, torch.float32), (128, 2, 20, torch.bfloat16),
                                      (64, 1, 100, torch.float16), (256, 1, 3, torch.float32), (256, 1, 30, torch.bfloat16)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_queries_that_are_not_finite_stay_by_themselves(cuda, D, H, n, od, bad):
    """Their rows are NaN, all others within the bounds that hold without them. (Not their bits: 32 rows that a warp of the kernel
    for many rows has go another way when one of them has such scores, fl(fl(s f) - base) for fl(s f - base). These are 2^-24 of the
    score apart at most, of the 2^-19 A that the bound has for scores.)"""
    from astc_kv_cuda import q4_attention
    cache, k, v = make(2, H, 700, D, seed=n, page=48)
    q = torch.randn(2, n, 4 * H, D, device="cuda").to(torch.bfloat16 if od != torch.float32 else od)
    lens = torch.tensor([700, 391], **i32)
    ref, _, A, vmax = plain_attention(q, k, v, [700, 391], [n, n], True, None)
    hit = torch.zeros(2, n, 4 * H, dtype=torch.bool, device="cuda")
    for b, t, h in ((0, 0, 1), (1, n - 1, 4 * H - 1)):
        q[b, t, h, (7 * h + t) % D] = bad
        hit[b, t, h] = True
    got = q4_attention(q, cache, lens, out_dtype=od).double()
    assert got[hit].isnan().all()
    tol = vmax * (2.0 ** -19 * A + 2.0 ** -18 + (2.0 ** -10 if od != torch.float32 else 0.0)) + HALF_ULP[od] * ref.abs() + 2.0 ** -25
    assert ((got - ref).abs() <= tol)[~hit].all()


@pytest.mark.parametrize("n", [1, 60])
def test_sequences_that_share_pages(cuda, n):
    from astc_kv_cuda import Q4Cache
    one, _, _ = make(1, 2, 400, 64, page=80, spare=6)
    table = one.block_table.repeat(3, 1)
    own = [p for p in range(one.k.shape[0]) if p not in one.block_table.flatten().tolist()]
    table[1, 3:], table[2, 2] = torch.tensor(own[:2], **i32), own[2]
    cache = Q4Cache(one.k, one.v, one.k_scales, one.v_scales, block_table=table)
    k, v = values_of(cache)
    q = torch.randn(3, n, 6, 64, device="cuda").bfloat16()
    check_attention(cache, k, v, q, [400, 399, 161], out_dtype=torch.bfloat16)
    check_attention(cache, k, v, q, [400, 399, 161])


def test_calls_at_the_same_time(cuda):
    """Three streams: two read one cache, one appends to another."""
    from astc_kv_cuda import Q4Append, Q4Attention, Q4Cache, Q4Restore, Rotary
    cache, _, _ = make(2, 4, 3000, 128, page=64)
    other = Q4Cache.zeros(2, 4, 3000, 128)
    lens = torch.tensor([3000, 1777], **i32)
    rot = Rotary.make(128, 3000)
    qkv = torch.randn(2, 200, 24, 128, device="cuda").bfloat16()
    calls = [Q4Attention(qkv[:, :n, :16], cache, lens, out_dtype=od) for n, od in ((1, torch.float32), (200, torch.bfloat16), (3, torch.bfloat16))]
    append = Q4Append(other, qkv[:, :, 16:20], qkv[:, :, 20:], torch.tensor([5, 900], **i32), rotary=rot, q=qkv[:, :, :16])
    back = Q4Restore(cache, None, 1000)
    want = [c.run().clone() for c in calls] + [append.run().clone(), other.k.clone(), *[t.clone() for t in back.run()]]
    torch.cuda.synchronize()
    for c in calls:
        c.out.zero_()
    for t in (append.q, other.k, other.v, other.k_scales, other.v_scales, back.k, back.v):
        t.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for s, group in zip(streams, (calls[:2], calls[2:] + [back], [append])):
            for c in group:
                c.run(s)
    torch.cuda.synchronize()
    got = [c.out for c in calls] + [append.q, other.k, back.k, back.v]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_out_on_top_of_the_queries_is_refused(cuda):
    from astc_kv_cuda import Q4Attention
    cache, _, _ = make(2, 2, 96, 64)
    q = torch.randn(2, 4, 64, device="cuda")
    with pytest.raises(ValueError):
        Q4Attention(q, cache, out=q)
    both = torch.randn(2, 2, 4, 64, device="cuda")
    with pytest.raises(ValueError):
        Q4Attention(both[:, 0], cache, out=both.view(4, 4, 64)[1:3])
    Q4Attention(both[0], cache, out=both[1]).run()


@pytest.mark.parametrize("interleaved", [False, True])
def test_backward_of_a_rotation_in_a_graph(cuda, interleaved):
    """Captured with its forward pass, replayed for other values: the gradients of the same passes run one by one."""
    from astc_kv_cuda import Rotary, rotate
    rot = Rotary.make(64, 50, sections=(12, 20), interleaved=interleaved)
    at = torch.randint(0, 50, (2, 3, 17), **i32)
    x = torch.randn(3, 17, 5, 96, device="cuda").requires_grad_()
    w = torch.randn(3, 17, 5, 96, device="cuda")

    def step():
        return torch.autograd.grad((rotate(x, rot, at) * w).square().sum(), x)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad = step()
    for _ in range(2):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            w.copy_(torch.randn_like(w))
            at.copy_(torch.randint_like(at, 0, 50))
        graph.replay()
        got = grad.clone()
        assert torch.equal(got, step())


@pytest.mark.parametrize("args", [["--prompt", "1500", "--steps", "5"], ["--prompt", "70", "--steps", "40", "--page", "16"]])
def test_the_example_runs(cuda, args):
    done = subprocess.run([sys.executable, str(Path(__file__).resolve().parents[1] / "examples" / "q4_serving.py"), *args],
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr
