"""More of the rotary positions on the GPU: derivatives of other kinds than the backward pass."""
import pytest
import torch
from torch.autograd import forward_ad

from test_gpu_rotary import TYPES, places_of, same, turned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", TYPES)
def test_tangents_are_rotated(cuda, dt, interleaved):
    from astc_kv_cuda import Rotary, rotate
    rot = Rotary.make(48, 30, sections=(8, 16), interleaved=interleaved)
    axes = [0] * 8 + [1] * 16
    at = places_of(2, 2, 5, 30, seed=3)
    x, v = (torch.randn(2, 5, 3, 64, device="cuda").to(dt) for _ in range(2))
    want = turned(v, rot.table, axes, at, interleaved)
    with forward_ad.dual_level():
        y = forward_ad.unpack_dual(rotate(forward_ad.make_dual(x, v), rot, at))
        same(y.primal, turned(x, rot.table, axes, at, interleaved))
        same(y.tangent, want)
    y, t = torch.func.jvp(lambda z: rotate(z, rot, at), (x,), (v,))
    same(t, want)
    # Along with a gradient: of the tangent's sum by the tangent.
    w = v.clone().requires_grad_()
    with forward_ad.dual_level():
        t = forward_ad.unpack_dual(rotate(forward_ad.make_dual(x, w), rot, at)).tangent
        same(torch.autograd.grad(t.sum(), w)[0], turned(torch.ones_like(v), rot.table, axes, at, interleaved, True))


def test_second_derivatives(cuda):
    """f = sum(y^3) / 3 of y = R x: the Hessian times v is R^T (2 y u) with u = R v. With X = |x1| + |x2| of a pair and V likewise,
    y is off by 2^-22 X, u by 2^-22 V, and eight more roundings make 2 y u off by 2 X V 2^-20; the last rotation adds up
    two of those and its own 2^-22 (4 X V): 2^-17 X V covers them."""
    from astc_kv_cuda import Rotary, rotate
    rot = Rotary.make(64, 30)
    at = places_of(1, 2, 5, 30)
    x, v = (torch.randn(2, 5, 3, 64, device="cuda") for _ in range(2))
    x.requires_grad_()
    g, = torch.autograd.grad((rotate(x, rot, at) ** 3).sum() / 3, x, create_graph=True)
    h, = torch.autograd.grad(g, x, v)

    def turn(z, inverse=False):
        return turned(z, rot.table, [0] * 32, at, False, inverse)
    y, u = turn(x.detach()), turn(v)
    want = turn((2 * y * u).float(), True)

    def size(z):
        z = z.detach().double().abs()
        return (z[..., :32] + z[..., 32:]).repeat(1, 1, 1, 2)
    assert ((h.double() - want).abs() <= 2.0 ** -17 * size(x) * size(v)).all()


def test_autograd_sees_what_is_written(cuda):
    """A rotation in place of what a backward pass needs is an error there, and one that would need a record is refused."""
    from astc_kv_cuda import Rotary, Rotate, rotate
    rot = Rotary.make(64, 30)
    at = places_of(1, 2, 5, 30)
    x = torch.randn(2, 5, 3, 64, device="cuda")
    w = torch.randn(64, device="cuda", requires_grad=True)
    for write in (lambda: rotate(x, rot, at, out=x), Rotate(x, rot, at, out=x).run):
        loss = (x * w).sum()  # keeps x
        write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    other, loss = x.clone(), (x * w).sum()
    Rotate(x, rot, at, out=other).run()
    loss.backward()
    y = torch.randn(2, 5, 3, 64, device="cuda", requires_grad=True) * 2
    before = y.detach().clone()
    call = Rotate(y, rot, at, out=y)
    for run in (call.run, lambda: rotate(x, rot, at, out=y)):
        with pytest.raises(ValueError):
            run()
    assert torch.equal(y, before)
    with forward_ad.dual_level():
        z = forward_ad.make_dual(x, x)
        with pytest.raises(ValueError):
            rotate(x.clone(), rot, at, out=z)
    # (What a transform does not look at stays as it is outside.)
    out = torch.empty_like(x)
    torch.func.grad(lambda s: (rotate(x, rot, at, out=out) * s).sum())(torch.ones(1, device="cuda"))
    same(out, turned(x, rot.table, [0] * 32, at, False))
    with torch.no_grad():
        call.run()
    same(y.detach(), turned(before, rot.table, [0] * 32, at, False))
    with torch.inference_mode():
        z = before.clone()
        rotate(z, rot, at, out=z)
    same(z, turned(before, rot.table, [0] * 32, at, False))


def test_learned_frequencies_are_refused(cuda):
    from astc_kv_cuda import Rotary, rotate
    f = torch.rand(32, device="cuda", requires_grad=True)
    at = places_of(1, 2, 5, 30)
    x = torch.randn(2, 5, 3, 64, device="cuda")
    for z in (x, x.clone().requires_grad_()):
        with pytest.raises(ValueError):
            rotate(z, Rotary.make(64, 30, frequencies=f), at)
        with torch.no_grad():
            rot = Rotary.make(64, 30, frequencies=f)
        same(rotate(z, rot, at).detach(), turned(x if z is x else z.detach(), rot.table, [0] * 32, at, False))


def test_outputs_that_overlap_themselves_are_refused(cuda):
    from astc_kv_cuda import Rotary, rotate
    rot = Rotary.make(64, 30)
    at = places_of(1, 2, 5, 30)
    x = torch.randn(2, 5, 3, 64, device="cuda")
    room = torch.zeros(4096, device="cuda")
    for stride in ((960, 192, 32, 1), (960, 96, 64, 1), (64, 192, 64, 1), (0, 192, 64, 1)):
        with pytest.raises(ValueError):
            rotate(x, rot, at, out=room.as_strided(x.shape, stride))
    for stride in ((960, 192, 64, 1), (192, 384, 64, 1), (64, 384, 128, 1)):
        same(rotate(x, rot, at, out=room.as_strided(x.shape, stride)), turned(x, rot.table, [0] * 32, at, False))
