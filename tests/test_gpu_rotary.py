"""Rotary positions on the GPU.

The definition rounds every product and every sum to fp32 and the result once
to the output's type: the plain implementation does each operation in 64 bits
(which hold a product of fp32 numbers exactly) and rounds it, and the kernel has
to give the same bits. Against the angle in 64 bits: a table entry is off by
half a step of fp32 (2^-25, entries are at most 1), products and sum by
half steps again: |y| errors stay below 2^-22 (|x1| + |x2|).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def turned(x, table, axes, places, interleaved, inverse=False):
    """x [B, n, H, D] rotated, as fp32 numbers in 64 bits; places [axes, B, n]."""
    pairs = table.shape[1]
    at = places.long()[torch.as_tensor(axes, device=x.device)]  # [pairs, B, n]
    cs = table.double()[at, torch.arange(pairs, device=x.device).view(-1, 1, 1)]
    c, s = (cs[..., i].permute(1, 2, 0)[:, :, None] for i in (0, 1))
    s = -s if inverse else s
    x = x.double()
    a, z = (x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]) if interleaved else (x[..., :pairs], x[..., pairs:2 * pairs])

    def f32(v):
        return v.float().double()
    y1, y2 = f32(f32(a * c) - f32(z * s)), f32(f32(z * c) + f32(a * s))
    y = torch.stack([y1, y2], -1).flatten(-2) if interleaved else torch.cat([y1, y2], -1)
    return torch.cat([y, x[..., 2 * pairs:]], -1)


def same(got, want):
    """Bit for bit, a NaN being a NaN."""
    want = want.float().to(got.dtype)
    assert got.shape == want.shape
    assert ((got == want) | (got.isnan() & want.isnan())).all()


def places_of(axes, B, n, P, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, P, (axes, B, n), generator=g, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("D,R,H,n", [(128, 128, 8, 33), (64, 64, 9, 7), (128, 64, 3, 5), (72, 72, 16, 11), (80, 80, 1, 1), (96, 48, 2, 19),
                                     (256, 256, 1, 6), (256, 32, 2, 3), (24, 16, 40, 2), (7, 6, 3, 5), (2, 2, 1, 1), (66, 34, 5, 9), (36, 12, 2, 4)])
def test_shapes(cuda, D, R, H, n, dt, interleaved):
    from astc_kv_cuda import Rotary, rotate
    rot = Rotary.make(R, 50, theta=100.0, interleaved=interleaved)
    x = torch.randn(2, n, H, D, device="cuda").to(dt)
    at = places_of(1, 2, n, 50)
    for inverse in (False, True):
        same(rotate(x, rot, at[0], inverse=inverse), turned(x, rot.table, [0] * (R // 2), at, interleaved, inverse))
    same(rotate(x, rot, at), turned(x, rot.table, [0] * (R // 2), at, interleaved))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R,sections", [(128, 128, (16, 24, 24)), (64, 64, (16, 16)), (128, 64, (1, 30, 1)), (72, 72, (0, 18, 18)),
                                          (40, 12, (1, 1, 1, 1, 1, 1)), (6, 6, (1, 1, 1))])
def test_axes(cuda, D, R, sections, interleaved):
    """Time, height and width, and other divisions of the pairs; an axis without pairs may hold any position."""
    from astc_kv_cuda import Rotary, rotate
    rot = Rotary.make(R, 40, sections=sections, interleaved=interleaved)
    assert rot.axis_count == len(sections)
    x = torch.randn(3, 17, 4, D, device="cuda").bfloat16()
    at = places_of(len(sections), 3, 17, 40, seed=R)
    axes = [a for a, m in enumerate(sections) for _ in range(m)]
    want = turned(x, rot.table, axes, at, interleaved)
    if 0 in sections:
        at[sections.index(0)] = 1 << 30
    same(rotate(x, rot, at), want)
    mixed = [i % len(sections) for i in range(R // 2)]  # the axes take turns
    rot = Rotary(rot.table, axes=mixed, interleaved=interleaved)
    at = places_of(len(sections), 3, 17, 40, seed=1)
    same(rotate(x, rot, at), turned(x, rot.table, mixed, at, interleaved))


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("D,R", [(128, 128), (64, 32), (20, 10)])
def test_strides_and_in_place(cuda, D, R, dt):
    """Slices of a fused projection, rows on odd elements, batches that share a row, results into slices, in place."""
    from astc_kv_cuda import Rotary, Rotate, rotate
    rot = Rotary.make(R, 64)
    at = places_of(1, 2, 9, 64, seed=3)
    axes = [0] * (R // 2)
    qkv = torch.randn(2, 9, 7, D, device="cuda").to(dt)
    q = qkv[:, :, 1:5]
    want = turned(q, rot.table, axes, at, False)
    same(rotate(q, rot, at[0]), want)
    odd = torch.randn(2, 9, 4, D + 3, device="cuda").to(dt)[..., 3:]
    same(rotate(odd, rot, at[0]), turned(odd, rot.table, axes, at, False))
    heads_first = torch.randn(2, 4, 9, D, device="cuda").to(dt).transpose(1, 2)
    same(rotate(heads_first, rot, at[0]), turned(heads_first, rot.table, axes, at, False))
    shared = q[:1].expand(2, 9, 4, D)
    same(rotate(shared, rot, at[0]), turned(shared, rot.table, axes, at, False))
    to = torch.full((2, 9, 6, D + 1), 7.0, device="cuda").to(dt)
    rotate(q, rot, at[0], out=to[:, :, 1:5, 1:])
    same(to[:, :, 1:5, 1:], want)
    assert (to[..., 0] == 7).all() and (to[:, :, 0] == 7).all() and (to[:, :, 5] == 7).all()
    before = qkv.clone()
    Rotate(q, rot, at[0], out=q).run()
    same(q, want)
    assert torch.equal(qkv[:, :, 0], before[:, :, 0]) and torch.equal(qkv[:, :, 5:], before[:, :, 5:])
    for out in (qkv[:, :, 2:6], q.as_strided(q.shape, q.stride(), q.storage_offset() + 1), shared):
        with pytest.raises(ValueError):
            Rotate(q, rot, at[0], out=out)


def test_far_positions(cuda):
    """Angles of positions past 2^17 are exact; scaling and frequencies of one's own."""
    from astc_kv_cuda import Rotary, rotate
    P, R = (1 << 17) + 5, 64
    f = torch.rand(R // 2, dtype=torch.float64, generator=torch.Generator().manual_seed(0)) * 3
    rot = Rotary.make(R, P, frequencies=f, scaling=1.25)
    x = torch.randn(1, 300, 2, R, device="cuda")
    at = torch.randint(P - 1000, P, (1, 300), device="cuda", dtype=torch.int32)
    a = at.double()[..., None, None] * f.cuda()
    x1, x2 = x[..., :R // 2].double(), x[..., R // 2:].double()
    want = 1.25 * torch.cat([x1 * a.cos() - x2 * a.sin(), x2 * a.cos() + x1 * a.sin()], -1)
    size = (x1.abs() + x2.abs()).repeat(1, 1, 1, 2)
    assert ((rotate(x, rot, at) - want).abs() <= 1.25 * 2.0 ** -22 * size).all()


@pytest.mark.parametrize("axes", [None, [0, 1] * 16])
def test_positions_outside_the_table(cuda, axes):
    from astc_kv_cuda import Rotary, rotate
    rot = Rotary(Rotary.make(64, 20).table, axes=axes)
    x = torch.randn(1, 6, 3, 80, device="cuda").half()
    A = rot.axis_count
    at = places_of(A, 1, 6, 20)
    want = turned(x, rot.table, axes or [0] * 32, at, False)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    rotate(x, rot, at, status=status)
    assert int(status) == 0
    for i, bad in enumerate((20, -1, 1 << 30, -(1 << 31))):
        at[i % A, 0, i] = bad
        want[0, i, :, :64] = float("nan")
    out = rotate(x, rot, at, status=status)
    same(out, want)
    assert int(status) == 1


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(cuda, dt, interleaved):
    """The gradient is the inverse rotation of the output's; against the formula, and (fp32) against differences."""
    from astc_kv_cuda import Rotary, rotate
    rot = Rotary.make(48, 30, sections=(8, 16), interleaved=interleaved)
    x = torch.randn(2, 5, 3, 64, device="cuda").to(dt).requires_grad_()
    at = places_of(2, 2, 5, 30, seed=2)
    w = torch.randn(2, 5, 3, 64, device="cuda").to(dt)
    y = rotate(x, rot, at)
    y.backward(w)
    axes = [0] * 8 + [1] * 16
    same(x.grad, turned(w, rot.table, axes, at, interleaved, True))
    got = torch.autograd.grad(rotate(x, rot, at).sum(), x)[0]  # a broadcast gradient
    same(got, turned(torch.ones_like(x), rot.table, axes, at, interleaved, True))
    if dt == torch.float32:
        # The map is linear: a difference quotient is off by the outputs' roundings alone, 2^-22 of the
        # values it is made of, over the step.
        step = 1.0
        g = torch.Generator(device="cuda").manual_seed(0)
        with torch.no_grad():
            for _ in range(20):
                v = torch.randn(x.shape, generator=g, device="cuda")
                up, down = rotate(x + step * v, rot, at).double(), rotate(x - step * v, rot, at).double()
                diff = ((up - down) / (2 * step) * w.double()).sum()
                bound = 2.0 ** -20 * ((x.abs() + step * v.abs()).double().sum() * w.double().abs().max())
                assert (diff - (x.grad.double() * v.double()).sum()).abs() <= bound
    with pytest.raises(ValueError):
        rotate(x, rot, at, out=torch.empty_like(x))


def test_back_and_forth(cuda):
    """The inverse of a rotation gives the input up to its roundings: 2^-22 of a pair's values each way, twice."""
    from astc_kv_cuda import Rotary, rotate
    rot = Rotary.make(128, 4096)
    x = torch.randn(2, 100, 5, 128, device="cuda")
    at = places_of(1, 2, 100, 4096)
    back = rotate(rotate(x, rot, at), rot, at, inverse=True)
    size = (x[..., :64].abs() + x[..., 64:].abs()).repeat(1, 1, 1, 2)
    assert ((back - x).abs() <= 2.0 ** -20 * size).all()


def test_values_that_are_not_finite(cuda):
    """They show in their own pairs and nowhere else."""
    from astc_kv_cuda import Rotary, rotate
    rot = Rotary.make(64, 10)
    x = torch.randn(1, 4, 2, 96, device="cuda").bfloat16()
    at = places_of(1, 1, 4, 10)
    x[0, 1, 0, 3], x[0, 2, 1, 40], x[0, 3, 0, 90] = float("nan"), float("inf"), float("nan")
    same(rotate(x, rot, at[0]), turned(x, rot.table, [0] * 32, at, False))


def test_empty_and_large(cuda):
    from astc_kv_cuda import Rotary, rotate
    rot = Rotary.make(64, 10)
    for shape in ((0, 3, 2, 64), (2, 0, 2, 64)):
        at = torch.zeros(shape[:2], dtype=torch.int32, device="cuda")
        assert rotate(torch.randn(shape, device="cuda"), rot, at).shape == shape
    # More than 2^31 elements, in place.
    rot = Rotary.make(128, 70000)
    x = torch.empty(1, 66000, 260, 128, device="cuda", dtype=torch.bfloat16)
    assert x.numel() > 1 << 31
    x.normal_()
    at = torch.randint(0, 70000, (1, 66000), device="cuda", dtype=torch.int32)
    tail = x[:, -3:].clone()
    rotate(x, rot, at, out=x)
    same(x[:, -3:], turned(tail, rot.table, [0] * 64, at[None, :, -3:], False))


def test_graph_streams_and_updates(cuda):
    """A captured call follows its positions and inputs; a call runs on another stream than the one it was built on."""
    from astc_kv_cuda import Rotary, Rotate
    rot = Rotary.make(64, 100)
    x = torch.randn(2, 3, 4, 64, device="cuda").half()
    at = places_of(1, 2, 3, 100)
    call = Rotate(x, rot, at)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call.run()
    side = torch.cuda.Stream()
    for seed in range(3):
        x.copy_(torch.randn(x.shape, device="cuda"))
        at.copy_(places_of(1, 2, 3, 100, seed))
        want = turned(x, rot.table, [0] * 32, at, False)
        call.out.zero_()
        graph.replay()
        same(call.out, want)
        call.out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        call.run(side)
        torch.cuda.current_stream().wait_stream(side)
        same(call.out, want)


def test_refusals(cuda):
    from astc_kv_cuda import Rotary, Rotate
    rot = Rotary.make(64, 10, sections=(16, 16))
    x = torch.randn(2, 3, 4, 64, device="cuda")
    at = places_of(2, 2, 3, 10)
    Rotate(x, rot, at)
    bad = [dict(positions=at[0]), dict(positions=at.long()), dict(positions=at[:, :, :2]), dict(positions=at[:, :1]), dict(x=x[0]),
           dict(x=x[..., :32]), dict(x=x.double()), dict(x=x.transpose(2, 3)), dict(x=torch.randn(2, 3, 4, 300, device="cuda")),
           dict(out=x.half()), dict(out=x[:1]), dict(out=x[..., :1].expand(2, 3, 4, 64)), dict(status=at.float()), dict(positions=at.cpu()),
           dict(x=x.cpu())]
    for kw in bad:
        with pytest.raises(ValueError):
            Rotate(**{"x": x, "rotary": rot, "positions": at, **kw})
    with pytest.raises(ValueError):
        Rotary(rot.table, axes=[0] * 31)
    with pytest.raises(ValueError):
        Rotary(rot.table, axes=[8] * 32)
    with pytest.raises(ValueError):
        Rotary(rot.table[:, 1:])
