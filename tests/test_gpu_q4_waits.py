"""Attention of many rows over the 4-bit cache whose bounded waits run out: with a limit of a few tries, microseconds,
CTAs give up here and there, as they would after seconds if something never came. What they
then write is NaN, whole rows of it, the status says so, and everything else is as without a limit."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TIMEOUT = 7


@pytest.mark.parametrize("od", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,H,G,n,T,split", [(64, 2, 1, 100, 2000, 0), (128, 2, 4, 30, 4096, 4096), (128, 4, 1, 300, 3000, 0),
                                             (128, 4, 4, 300, 4096, 4096), (64, 4, 3, 509, 2000, 2048), (256, 2, 1, 300, 2000, 2048),
                                             (256, 1, 2, 200, 4000, 0), (128, 4, 1, 300, 16384, 16384)])
def test_rows_that_were_given_up_are_nan(cuda, D, H, G, n, T, split, od):
    from astc_kv_cuda import Q4Attention, Q4Cache
    from test_gpu_q4 import make
    c, _, _ = make(2, H, T, D, seed=D + n)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = Q4Cache(c.k, c.v, c.k_scales, c.v_scales, max_tokens=T, status=status)
    q = torch.randn(2, n, H * G, D, device="cuda").to(od)
    lens = torch.tensor([T, T // 2], dtype=torch.int32, device="cuda")
    call = Q4Attention(q, cache, lens, out_dtype=od, lse=True, split_tokens=split)
    want, lse = call.run().clone(), call.lse.clone()
    assert int(status) == 0 and not want.isnan().any()
    for tries in (1, 2, 3, 4, 6, 9, 1 << 22):
        status.zero_()
        call.desc.wait_tries = tries
        call.out.fill_(1.0)
        call.lse.fill_(1.0)
        out = call.run()
        gone = out.isnan().any(-1)
        assert out[gone].isnan().all() and torch.equal(out[~gone], want[~gone])
        assert call.lse[gone].isnan().all() and torch.equal(call.lse[~gone], lse[~gone])
        assert int(status) == TIMEOUT or not gone.any() and int(status) == 0
        # The longest case's last 44 rows are half a CTA, whose other half waits from the beginning to the end, 200 us.
        assert T < 16384 or tries > 1 or gone.any()
    assert int(status) == 0 and not gone.any()
