"""Rotary positions on the GPU: text, images (height and width), video (time,
height and width).

A `Rotary` holds the cosines and sines of every position, made once in 64
bits. `Rotate` turns the heads of tokens by them, `Q4Append` (q4.py) turns keys
and queries on their way into the 4-bit cache. The gradient of a rotation is
the inverse rotation of the output's gradient: `Rotate(..., inverse=True)`, and
`rotate` records it.

The calls follow `Q8Attention`: an object that checks its tensors and builds
its C descriptor once and is re-issued with `run()`. Everything below runs in
libakv_cuda.so (C ABI: include/akv_rotary.h, which has the formulas).
"""
from __future__ import annotations

from collections.abc import Sequence
from dataclasses import dataclass

import torch
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.graph import increment_version

from . import _lib as L
from .q8 import _DTYPES, _Call, _int32, _may_overlap, _on, _rows


@dataclass(eq=False)
class Rotary:
    """Positions and the pairs that they turn.

    `table` fp32 [positions, pairs, 2]: cosine and sine of each pair at each
    position. Pairs are channels (i, i + pairs), or (2i, 2i + 1) when
    `interleaved`; a head's channels from 2 * pairs on stay. `axes`: for each
    pair the axis (from 0) whose position it takes, None for one axis.
    """
    table: torch.Tensor
    axes: Sequence[int] | None = None
    interleaved: bool = False

    def __post_init__(self):
        t = self.table
        if t.dim() != 3 or t.shape[2] != 2 or t.dtype != torch.float32 or not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError("table must be contiguous fp32 [positions, pairs, 2], 16-byte aligned")
        if not t.is_cuda:
            raise ValueError("expected CUDA tensors")
        if not 1 <= t.shape[1] <= 128 or not 1 <= t.shape[0] < 1 << 31:
            raise ValueError("a table has 1 to 128 pairs and a position at least")
        axes = [0] * self.pairs if self.axes is None else [int(a) for a in self.axes]
        if len(axes) != self.pairs or not all(0 <= a < L.AKV_ROTARY_MAX_AXES for a in axes):
            raise ValueError(f"axes must name an axis below {L.AKV_ROTARY_MAX_AXES} for each pair")
        self.axis_count = max(axes) + 1
        c = L.AkvRotary()
        c.table_dev, c.positions, c.rotary_dim = t.data_ptr(), t.shape[0], 2 * self.pairs
        c.axes, c.interleaved = self.axis_count, int(self.interleaved)
        c.axis[:self.pairs] = axes
        self._c = c

    @classmethod
    def make(cls, rotary_dim: int, positions: int, *, theta: float = 10000.0, frequencies: torch.Tensor | None = None,
             scaling: float = 1.0, sections: Sequence[int] | None = None, axes: Sequence[int] | None = None, interleaved: bool = False,
             device: torch.device | str = "cuda") -> "Rotary":
        """The table of angles p * frequencies[i] (default: theta^(-2 i / rotary_dim)) for p < positions, in 64 bits, times
        `scaling`. `sections`: how many consecutive pairs take axis 0, 1, ...; or `axes` as above."""
        if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > 256:
            raise ValueError("rotary_dim must be even, 2 to 256")
        if positions < 1:
            raise ValueError("positions must be positive")
        pairs = rotary_dim // 2
        if frequencies is None:
            frequencies = theta ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
        if tuple(frequencies.shape) != (pairs,):
            raise ValueError("frequencies must be one for each pair")
        if sections is not None:
            if axes is not None or sum(sections) != pairs or any(n < 0 for n in sections):
                raise ValueError("sections must add up to the pairs (and stand in axes' place)")
            axes = [a for a, n in enumerate(sections) for _ in range(n)]
        angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * frequencies.to(device=device, dtype=torch.float64)
        table = torch.stack([angle.cos(), angle.sin()], -1).mul_(scaling).float()
        return cls(table, axes=axes, interleaved=interleaved)

    @property
    def device(self) -> torch.device:
        return self.table.device

    @property
    def pairs(self) -> int:
        return self.table.shape[1]

    def _places(self, positions: torch.Tensor, batch: int, n: int) -> int:
        """Address of positions [batch, n] (one axis) or [axes, batch, n]."""
        shape = (self.axis_count, batch, n)
        return _int32("positions", positions, shape[1:] if positions.dim() == 2 and self.axis_count == 1 else shape)


def _overlaps_itself(t: torch.Tensor) -> bool:
    """Whether two elements of a tensor are at one place."""
    if t.numel() == 0:
        return False
    dims = sorted([(s, n) for s, n in zip(t.stride(), t.shape) if n > 1], reverse=True)
    extent = 1
    for s, n in reversed(dims):  # nested, as most are?
        if s < extent:
            break
        extent += s * (n - 1)
    else:
        return False

    def meet(left: int, dims: list) -> bool:
        # Is left = sum of s * i with -n < i < n?
        if not dims:
            return left == 0
        (s, n), span = dims[0], sum(r * (m - 1) for r, m in dims[1:])
        if abs(left) > span + s * (n - 1) or s == 0:
            return left == 0
        return any(meet(left - s * i, dims[1:]) for i in range(max(-(-(left - span) // s), 1 - n), min((left + span) // s, n - 1) + 1))

    for k, (s, n) in enumerate(dims):
        rest = dims[k + 1:]
        if s == 0 or any(meet(s * i, rest) for i in range(1, min(n - 1, sum(r * (m - 1) for r, m in rest) // s) + 1)):
            return True
    return False


class Rotate(_Call):
    """Rotate x [B, n, H, D] at `positions` int32 [B, n], or [axes, B, n] with
    several axes, read when the call runs. x may be a strided view, for example
    the queries and keys of a fused projection. `out`: x itself (in place), or
    a tensor that does not overlap it; its own contiguous one by default.
    `inverse`: turns back, which is the gradient. A token with a position
    outside the table becomes NaN in the rotated channels, and `status`
    (optional int32 [1]) gets an error code. Records no gradient (see `rotate`):
    an `out` that requires one is refused where gradients are recorded, and
    autograd learns that a given `out` was written."""

    _family, _fn = "", "rotate"

    def __init__(self, x: torch.Tensor, rotary: Rotary, positions: torch.Tensor, *, out: torch.Tensor | None = None,
                 inverse: bool = False, status: torch.Tensor | None = None):
        if x.dim() != 4:
            raise ValueError("x must be [B, n, H, D]")
        if not x.is_cuda:
            raise ValueError("expected CUDA tensors")
        _on(x.device, table=rotary.table, positions=positions, out=out, status=status)
        B, n, H, D = x.shape
        if 2 * rotary.pairs > D or D > 256 or H < 1:
            raise ValueError("heads need as many channels as the pairs have, and at most 256")
        if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
            raise ValueError("status must be int32")
        self._given = out is not None
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if out.dtype != x.dtype:
            raise ValueError("out must have the dtype of x")
        d = L.AkvRotateDesc()
        d.rotary = rotary._c
        d.batch, d.tokens, d.heads, d.head_dim, d.inverse = B, n, H, D, int(inverse)
        d.x_dev, d.x_stride[:] = _rows("x", x, (B, n, H, D))
        d.out_dev, d.out_stride[:] = _rows("out", out, (B, n, H, D))
        d.dtype = _DTYPES[x.dtype]
        same = d.x_dev == d.out_dev and all(a == b or s < 2 for a, b, s in zip(x.stride(), out.stride(), x.shape))
        if not same and _may_overlap(x, out):
            raise ValueError("out must be x or not overlap it")
        if self._given and _overlaps_itself(out):
            raise ValueError("out must not have two elements at one place")
        d.positions_dev = rotary._places(positions, B, n)
        d.status_dev = None if status is None else status.data_ptr()
        self.out = out
        self._prepare(d, x.device, x, out, rotary.table, positions, status)

    def run(self, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        if self._given:
            if _derived(self.out):
                raise ValueError("a rotation into a given tensor records no gradient or tangent, which this one has")
            increment_version(self.out)
        self._issue(stream)
        return self.out


class _Rotation(torch.autograd.Function):
    """A rotation is linear: both of its derivatives are rotations of the same positions, recorded where they are needed again."""

    @staticmethod
    def forward(x, rotary, positions, inverse):
        return Rotate(x, rotary, positions, inverse=inverse).run()

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, ctx.rotary, positions, ctx.inverse = inputs
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)

    @staticmethod
    def backward(ctx, grad):
        return rotate(_contiguous(grad), ctx.rotary, ctx.saved_tensors[0], inverse=not ctx.inverse), None, None, None

    @staticmethod
    def jvp(ctx, tangent, *_):
        return rotate(_contiguous(tangent), ctx.rotary, ctx.saved_tensors[0], inverse=ctx.inverse)


def _contiguous(x: torch.Tensor) -> torch.Tensor:
    # (A broadcast gradient, of a sum for example, has no contiguous last dimension.)
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


# Whether a transform of torch.func is at work.
_transforming = getattr(torch._C, "_are_functorch_transforms_active", lambda: False)


def _derived(x: torch.Tensor) -> bool:
    """Whether a derivative by x is recorded, backward or forward."""
    return x.requires_grad and torch.is_grad_enabled() or unpack_dual(x).tangent is not None


def rotate(x: torch.Tensor, rotary: Rotary, positions: torch.Tensor, *, inverse: bool = False, stream: torch.cuda.Stream | None = None,
           **kw) -> torch.Tensor:
    """One `Rotate`; x may require a gradient or have a tangent (on the current stream, without out). As with any operation of
    autograd, a backward pass is captured into a CUDA graph only while no graph recorded outside the capture holds the same leaves.
    The table gets no gradient: one that requires it is refused."""
    if _derived(rotary.table):
        raise ValueError("the rotary table takes no gradient")
    if _derived(x) or _transforming() and stream is None and not kw:
        if stream is not None or kw:
            raise ValueError("a rotation that records a gradient runs on the current stream and takes no out or status")
        return _Rotation.apply(x, rotary, positions, inverse)
    return Rotate(x, rotary, positions, inverse=inverse, **kw).run(stream)
