"""Codes in the 4-bit cache, every bit of them: the signs of zeros too."""
import pytest
import torch

from test_gpu_q4 import TYPES, quantised
from test_gpu_rotary import turned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rotated", [False, True])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("D,n", [(128, 3), (128, 140), (64, 140), (96, 5), (256, 140), (32, 9)])
def test_signs_of_zeros(cuda, D, n, dt, rotated):
    """A group with a scale of 0 has codes of 0, whatever its values' signs (below 2^-25 x 6 the scale is 0 in fp16, which all three
    types hold some of); where the scale is a number, what rounds to 0 keeps its sign."""
    from astc_kv_cuda import Q4Append, Q4Cache, Rotary
    g = torch.Generator(device="cuda").manual_seed(D + n)
    k, v = (torch.randn(1, n, 2, D, generator=g, device="cuda") for _ in range(2))
    tiny = torch.rand(1, n, 2, D // 32, 1, generator=g, device="cuda") < 0.4
    tiny[:, 0] = True
    # (After a rotation, too: no value grows by more than the root of 2.)
    k, v = (torch.where(tiny, x.unflatten(-1, (-1, 32)).sign() * 2.0 ** -24, x.unflatten(-1, (-1, 32))).flatten(-2).to(dt) for x in (k, v))
    rot = Rotary.make(D, n) if rotated else None
    cache = Q4Cache.zeros(1, 2, n, D)
    cache.k.fill_(0xFF)
    cache.v.fill_(0xFF)
    Q4Append(cache, k, v, torch.zeros(1, dtype=torch.int32, device="cuda"), rotary=rot).run()
    at = torch.arange(n, device="cuda").view(1, 1, n)
    for codes, scales, x in ((cache.k, cache.k_scales, turned(k, rot.table, [0] * (D // 2), at, False) if rotated else k.double()),
                             (cache.v, cache.v_scales, v.double())):
        wc, ws = quantised(x)
        wc = torch.where(ws[..., None] > 0, wc.unflatten(-1, (-1, 16)), 0).flatten(-2)
        assert (ws == 0).any() and ((wc & 15) == 8).any()
        assert torch.equal(scales[..., :n], ws.permute(0, 2, 3, 1))
        assert torch.equal(codes[:, :, :n], wc.transpose(1, 2))
