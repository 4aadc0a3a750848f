"""`rotate` and derivatives, without a GPU: a plain rotation stands in for the call, and the recording around it is checked."""
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad

from astc_kv_cuda import rotary


class Plain:
    """What Rotate does, in 64 bits and without a record."""

    def __init__(self, x, table, positions, *, inverse=False, out=None):
        x.data_ptr()  # as Rotate: memory, or an error
        cs = table.table[positions.long()][:, :, None]
        c, s = cs[..., 0], cs[..., 1] * (-1 if inverse else 1)
        a, b = x.detach().chunk(2, -1)
        self.out = torch.cat([a * c - b * s, b * c + a * s], -1)

    def run(self, stream=None):
        return self.out


@pytest.fixture
def given(monkeypatch):
    monkeypatch.setattr(rotary, "Rotate", Plain)
    g = torch.Generator().manual_seed(0)
    angle = torch.randn(9, 3, dtype=torch.float64, generator=g)
    table = torch.stack([angle.cos(), angle.sin()], -1) * 1.5
    x, v = torch.randn(2, 2, 4, 2, 6, dtype=torch.float64, generator=g)
    return x, v, SimpleNamespace(table=table), torch.randint(0, 9, (2, 4), generator=g)


def test_tangents_are_rotated(given):
    x, v, table, at = given
    want = Plain(v, table, at).run()
    with forward_ad.dual_level():
        y = rotary.rotate(forward_ad.make_dual(x, v), table, at)
        assert torch.equal(forward_ad.unpack_dual(y).tangent, want)
        y = rotary.rotate(forward_ad.make_dual(x, v[..., :1].expand_as(v)), table, at)  # broadcast
        assert torch.equal(forward_ad.unpack_dual(y).tangent, Plain(v[..., :1].expand_as(v), table, at).run())
    assert torch.equal(torch.func.jvp(lambda z: rotary.rotate(z, table, at), (x,), (v,))[1], want)


@pytest.mark.parametrize("inverse", [False, True])
def test_derivatives_of_any_order(given, inverse):
    x, _, table, at = given
    x = x.requires_grad_()
    assert torch.autograd.gradcheck(lambda z: rotary.rotate(z, table, at, inverse=inverse), x, check_forward_ad=True)
    assert torch.autograd.gradgradcheck(lambda z: rotary.rotate(z, table, at, inverse=inverse).sin(), x, check_fwd_over_rev=True)


def test_transforms(given):
    x, v, table, at = given

    def f(z):
        return rotary.rotate(z, table, at).sin().sum()
    leaf = x.clone().requires_grad_()
    g, = torch.autograd.grad(f(leaf), leaf, create_graph=True)
    assert torch.equal(torch.func.grad(f)(x), g)
    h, = torch.autograd.grad(g, leaf, v)
    assert torch.allclose(torch.func.jvp(torch.func.grad(f), (x,), (v,))[1], h, rtol=1e-12)
    with pytest.raises(RuntimeError):
        torch.func.vmap(f)(x[None])


def test_a_table_that_requires_a_gradient(given):
    x, v, rot, at = given
    learned = SimpleNamespace(table=rot.table.clone().requires_grad_())
    with pytest.raises(ValueError):
        rotary.rotate(x, learned, at)
    with torch.no_grad():
        assert torch.equal(rotary.rotate(x, learned, at), rotary.rotate(x, rot, at))
    with forward_ad.dual_level(), pytest.raises(ValueError):
        rotary.rotate(x, SimpleNamespace(table=forward_ad.make_dual(rot.table, rot.table)), at)


@pytest.mark.parametrize("shape,stride,overlaps", [
    ((2, 3, 4, 8), (96, 32, 8, 1), False), ((2, 3, 4, 8), (96, 32, 0, 1), True), ((2, 3, 1, 8), (96, 32, 0, 1), False), ((2, 3, 4, 8), (8, 16, 48, 1), False),
    ((1, 3, 2, 32), (7, 64, 96, 1), False), ((1, 3, 2, 32), (7, 64, 80, 1), True), ((1, 9, 2, 32), (7, 16, 144, 1), True), ((2, 9, 2, 32), (1, 64, 1000, 2), False),
    ((2, 9, 2, 32), (31, 64, 1000, 1), True), ((0, 3, 4, 8), (0, 0, 0, 1), False), ((2, 2, 2, 2), (4, 2, 3, 1), True), ((1, 1, 1, 1), (0, 0, 0, 0), False),
    ((3, 100000, 64, 128), (819200000, 8192, 128, 1), False), ((3, 100000, 64, 128), (819199999, 8192, 128, 1), True),
    ((3, 100000, 64, 128), (128, 24576, 384, 1), False)])
def test_an_output_that_overlaps_itself(shape, stride, overlaps):
    t = torch.empty(1, dtype=torch.bfloat16, device="meta").as_strided(shape, stride)
    assert rotary._overlaps_itself(t) == overlaps
    if t.numel() < 10000:
        places = sum(torch.arange(n).mul(s).view([-1 if i == k else 1 for i in range(4)]) for k, (n, s) in enumerate(zip(shape, stride)))
        assert (places.unique().numel() < t.numel()) == overlaps
