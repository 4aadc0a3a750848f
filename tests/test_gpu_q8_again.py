"""Calls on the 8-bit cache that are prepared once and run again, on other
streams, and in memory that they share."""
import ctypes as ct

import pytest
import torch

from test_gpu_q8 import make, plain_choice

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
