"""The 8-bit KV cache: store, attention, eviction, restore on the GPU.

A `Q8Cache` holds K and V as int8 or e4m3 codes with one fp32 scale for every
block of tokens of a kv head (value = code * scale), in one piece or in pages
found through a block table. The calls follow `ops.Attention`: an object that
checks its tensors, builds the C descriptor and its workspace once and is
re-issued with `run()`, and a function for a single call.

* `Q8Store` quantises new tokens into the cache,
* `Q8Attention` attends one or many new tokens per sequence to it and can add
  up the attention weight that every cached token receives,
* `Q8Evict` packs the tokens with the largest accumulated weight into a
  smaller cache,
* `Q8Restore` returns tokens as values.

Lengths, positions and block tables are int32 CUDA tensors that are read when
a call runs, so a program updates them in place between steps. A call's
outputs and workspace are its own and written anew by every run: runs of one
call follow one another, on one stream or on streams that the program orders.
Everything
below runs in libakv_cuda.so (C ABI: include/akv_q8.h, which has the formulas
and the rules for empty rows, ties and values that are not finite).
"""
from __future__ import annotations

import ctypes as ct
from dataclasses import dataclass

import torch

from . import _lib as L

_DTYPES = {torch.float32: L.AKV_Q_F32, torch.bfloat16: L.AKV_Q_BF16, torch.float16: L.AKV_Q_F16}
_FORMATS = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


# The current stream's handle without building a Stream object (3 us a call).
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _on(device: torch.device, **tensors: torch.Tensor | None) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} must be on {device}")


def _int32(name: str, t: torch.Tensor | None, shape: tuple) -> int | None:
    """Address of an int32 tensor that a kernel reads in place."""
    if t is None:
        return None
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 {list(shape)}")
    return t.data_ptr()


def _rows(name: str, t: torch.Tensor, shape: tuple) -> tuple:
    """(address, batch / token / head strides) of [B, n, H, D] rows with contiguous head dimensions."""
    if t.dtype not in _DTYPES or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be fp32/bf16/fp16 {list(shape)}")
    if shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have a contiguous last dimension")
    return t.data_ptr(), t.stride()[:3]


@dataclass(eq=False)
class Q8Cache:
    """K and V codes with their scales.

    One piece: codes [B, H, T, D], scales [B, H, ceil(T / block_tokens)].
    Paged: codes [num_pages, H, page_tokens, D], scales [num_pages, H,
    page_tokens / block_tokens] and `block_table` int32 [B, pages_per_seq].
    The codes' dtype (int8 or float8_e4m3fn) is the format. Codes may be
    views whose last dimension is contiguous and whose other strides are
    multiples of 16 bytes. `max_tokens` (default: all there is room for)
    bounds a sequence. `status`: optional int32 [1] that kernels write an
    error code to (a bad table entry, a store past the end, a wait inside a
    kernel that ran out); without it such rows are dropped or read as zeros
    and nothing says so.
    """
    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor
    block_tokens: int = 64
    block_table: torch.Tensor | None = None
    max_tokens: int = 0
    status: torch.Tensor | None = None

    def __post_init__(self):
        if self.k.dim() != 4 or self.k.dtype not in _FORMATS.values():
            raise ValueError("codes must be int8 or float8_e4m3fn [pages or B, H, tokens, D]")
        if not self.k.is_cuda:
            raise ValueError("expected CUDA tensors")
        if self.v.shape != self.k.shape or self.v.dtype != self.k.dtype:
            raise ValueError("K and V codes must have the same shape and dtype")
        n, h, rows, d = self.k.shape
        if self.block_tokens not in (16, 32, 64, 128):
            raise ValueError("block_tokens must be 16, 32, 64 or 128")
        if d % 16 or not 16 <= d <= 256:
            raise ValueError("head_dim must be a multiple of 16, at most 256")
        if rows < 1 or h < 1:
            raise ValueError("a cache needs tokens and heads")
        blocks = -(-rows // self.block_tokens)
        for name in ("k", "v"):
            codes, scales = getattr(self, name), getattr(self, name + "_scales")
            if codes.stride(-1) != 1 or any(s % 16 for s in codes.stride()[:-1]) or codes.data_ptr() % 16:
                raise ValueError("codes need a contiguous last dimension, other strides in multiples of 16 bytes and 16-byte alignment")
            if scales.dtype != torch.float32 or tuple(scales.shape) != (n, h, blocks) or (blocks > 1 and scales.stride(-1) != 1):
                raise ValueError(f"scales must be fp32 {[n, h, blocks]} with a contiguous last dimension")
        _on(self.device, v=self.v, k_scales=self.k_scales, v_scales=self.v_scales, block_table=self.block_table, status=self.status)
        if self.status is not None and (self.status.dtype != torch.int32 or self.status.numel() < 1):
            raise ValueError("status must be int32")
        if self.block_table is None:
            self.batch, room = n, rows
        else:
            if rows % self.block_tokens:
                raise ValueError("a page must hold whole blocks")
            if self.block_table.dim() != 2:
                raise ValueError("block_table must be [B, pages_per_seq]")
            _int32("block_table", self.block_table, tuple(self.block_table.shape))
            self.batch, room = self.block_table.shape[0], self.block_table.shape[1] * rows
        self.max_tokens = self.max_tokens or room
        if not 0 < self.max_tokens <= room:
            raise ValueError("max_tokens exceeds what the cache has room for")
        c = L.AkvQ8Cache()
        c.format = L.AKV_Q8_INT8 if self.k.dtype == torch.int8 else L.AKV_Q8_E4M3
        c.block_tokens, c.batch, c.kv_heads, c.head_dim = self.block_tokens, self.batch, h, d
        c.max_tokens = self.max_tokens
        c.page_tokens = blocks * self.block_tokens if self.block_table is None else rows
        if self.block_table is not None:
            c.block_table_dev = self.block_table.data_ptr()
            c.pages_per_seq, c.num_pages = self.block_table.shape[1], n
        for name in ("k", "v"):
            codes, scales, side = getattr(self, name), getattr(self, name + "_scales"), L.AkvQ8Side()
            first, head = (codes.stride(0), codes.stride(1)), (scales.stride(0), scales.stride(1))
            side.codes, side.scales, side.stride_token = codes.data_ptr(), scales.data_ptr(), codes.stride(2)
            side.stride_head, side.scale_stride_head = first[1], head[1]
            if self.block_table is None:
                side.stride_batch, side.scale_stride_batch = first[0], head[0]
            else:
                side.stride_page, side.scale_stride_page = first[0], head[0]
            setattr(c, name, side)
        c.status_dev = None if self.status is None else self.status.data_ptr()
        self._c = c

    @classmethod
    def zeros(cls, batch: int, kv_heads: int, max_tokens: int, head_dim: int, *, fmt: str = "int8", block_tokens: int = 64,
              page_tokens: int = 0, block_table: torch.Tensor | None = None, num_pages: int = 0,
              status: torch.Tensor | None = None, device: torch.device | str = "cuda") -> "Q8Cache":
        """An empty cache: in one piece, or `num_pages` pages of `page_tokens` for a block table."""
        if fmt not in _FORMATS:
            raise ValueError("fmt must be 'int8' or 'fp8'")
        if block_tokens <= 0:
            raise ValueError("block_tokens must be 16, 32, 64 or 128")
        if block_table is None:
            n, rows = batch, -(-max_tokens // block_tokens) * block_tokens
        else:
            n, rows = num_pages, page_tokens
        def codes():
            return torch.zeros(n, kv_heads, rows, head_dim, dtype=torch.int8, device=device).view(_FORMATS[fmt])
        def scales():
            return torch.zeros(n, kv_heads, -(-rows // block_tokens), dtype=torch.float32, device=device)
        return cls(codes(), codes(), scales(), scales(), block_tokens=block_tokens, block_table=block_table, max_tokens=max_tokens,
                   status=status)

    @property
    def device(self) -> torch.device:
        return self.k.device

    @property
    def kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3]

    @property
    def fmt(self) -> str:
        return "int8" if self.k.dtype == torch.int8 else "fp8"

    @property
    def nbytes(self) -> int:
        """Resident bytes: codes and scales."""
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scales, self.v_scales))


class _Call:
    """A prepared call (of the 8-bit cache, the 4-bit cache or the rotation): a C descriptor, the tensors it points to, and `_issue`.

    Outputs and workspace are the object's own, so its runs follow one another
    on one stream, or on streams that the caller orders. The first run on
    another stream than the one the object was built on waits for what that
    one has been given so far: earlier work on the memory that the object took.
    """

    _family, _fn = "q8_", ""

    def _prepare(self, desc, device: torch.device, *tensors) -> None:
        self.desc, self.device = desc, device
        self._dref = ct.byref(desc)
        self._index = device.index if device.index is not None else 0
        self._tensors = [t for t in tensors if t is not None]
        self._issue_c = getattr(L.lib(), "akv_" + self._family + self._fn)
        self._home, self._met = _current_stream(self._index), set()

    def _issue(self, stream: torch.cuda.Stream | None) -> None:
        if torch.cuda.current_device() != self._index:
            raise ValueError(f"the tensors are on {self.device}, which is not the current device")
        handle = _current_stream(self._index) if stream is None else stream.cuda_stream
        if handle != self._home:
            self._elsewhere(handle, torch.cuda.current_stream(self._index) if stream is None else stream)
        code = self._issue_c(self._dref, handle or None)
        if code:
            raise L.AkvError(code, self._family + self._fn)

    def _elsewhere(self, handle: int, stream: torch.cuda.Stream) -> None:
        """Before a run on another stream than the one the object was built on."""
        # (A capture waits for all streams before it begins.)
        if handle not in self._met:
            home = torch.cuda.ExternalStream(self._home, self.device) if self._home else torch.cuda.default_stream(self.device)
            if not _capturing(stream) and not _capturing(home):
                stream.wait_stream(home)
                self._met.add(handle)
        # The caller may drop this object while the stream still works on its memory.
        for t in self._tensors:
            t.record_stream(stream)


class Q8Store(_Call):
    """Quantise k, v [B, n, H, D] into tokens start[b] .. start[b] + counts[b] - 1
    (n each without counts) of `cache`. Rows may be strided views, for example
    slices of a fused projection."""

    _fn = "store"

    def __init__(self, cache: Q8Cache, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor,
                 counts: torch.Tensor | None = None):
        if k.dim() != 4:
            raise ValueError("k must be [B, n, H, D]")
        _on(cache.device, k=k, v=v, start=start, counts=counts)
        if start is None or k.dtype != v.dtype:
            raise ValueError("start is needed, and k and v must have one dtype")
        d = L.AkvQ8StoreDesc()
        d.cache, d.tokens = cache._c, k.shape[1]
        shape = (cache.batch, k.shape[1], cache.kv_heads, cache.head_dim)
        d.k_dev, d.k_stride[:] = _rows("k", k, shape)
        d.v_dev, d.v_stride[:] = _rows("v", v, shape)
        d.dtype = _DTYPES[k.dtype]
        d.start_dev = _int32("start", start, (cache.batch,))
        d.counts_dev = _int32("counts", counts, (cache.batch,))
        self.cache = cache
        self._prepare(d, cache.device, k, v, start, counts, *_cache_tensors(cache))

    def run(self, stream: torch.cuda.Stream | None = None) -> Q8Cache:
        self._issue(stream)
        return self.cache


class Q8Restore(_Call):
    """Tokens start[b] + i (i without start), i < count, as values: (k, v) [B, count, H, D]."""

    _fn = "restore"

    def __init__(self, cache: Q8Cache, start: torch.Tensor | None, count: int, dtype: torch.dtype = torch.float32):
        if dtype not in _DTYPES:
            raise ValueError("dtype must be fp32, bf16 or fp16")
        if count < 0:
            raise ValueError("count must not be negative")
        _on(cache.device, start=start)
        shape = (cache.batch, count, cache.kv_heads, cache.head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=cache.device)
        self.v = torch.empty(shape, dtype=dtype, device=cache.device)
        d = L.AkvQ8RestoreDesc()
        d.cache, d.tokens, d.dtype = cache._c, count, _DTYPES[dtype]
        d.start_dev = _int32("start", start, (cache.batch,))
        d.k_dev, d.v_dev = self.k.data_ptr(), self.v.data_ptr()
        self._prepare(d, cache.device, self.k, self.v, start, *_cache_tensors(cache))

    def run(self, stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        self._issue(stream)
        return self.k, self.v


class Q8Attention(_Call):
    """Attention of the newest tokens of each sequence over the cache.

    q: [B, Hq, D] (one token per sequence) or [B, n, Hq, D], strided views
    allowed. `lens` int32 [B]: cached tokens per sequence, the queries' own
    included (None: the cache's max_tokens). `q_lens` int32 [B]: queries per
    sequence out of n (the rest of the output is zero). `causal`: query i sees
    tokens up to its own; otherwise every query sees the whole sequence.
    `out_dtype` fp32 (default) or a 16-bit type, which also lets the softmax
    weights meet V as fp16. `lse=True` keeps ln sum exp of the scores in
    `self.lse` [B, n, Hq]. `weights` fp32 [B, H, >= max_tokens]: the softmax
    weight each token received, over the queries and the kv head's query
    heads, is added to it (`accumulate=False`: replaces it).

    Splits and workspace go by the cache's max_tokens, not by the lengths; with
    `weights` and up to 16 rows (queries x heads of a kv head; 8 above head_dim
    128) the workspace holds 4 bytes per row, kv head and token of it. Where a
    cache has much more room than tokens, a second Q8Cache over the same tensors
    with a smaller `max_tokens` serves it faster.
    """

    _fn = "attention"

    def __init__(self, q: torch.Tensor, cache: Q8Cache, lens: torch.Tensor | None = None, *, q_lens: torch.Tensor | None = None,
                 causal: bool = True, scale: float = 0.0, out: torch.Tensor | None = None,
                 out_dtype: torch.dtype = torch.float32, lse: bool = False, weights: torch.Tensor | None = None,
                 accumulate: bool = True, split_tokens: int = 0):
        if q.dim() not in (3, 4):
            raise ValueError("q must be [B, Hq, D] or [B, n, Hq, D]")
        _on(cache.device, q=q, lens=lens, q_lens=q_lens, out=out, weights=weights)
        rows = q if q.dim() == 4 else q.unsqueeze(1)
        B, n, Hq, D = rows.shape
        d = L.AkvQ8AttnDesc()
        d.cache = cache._c
        if Hq == 0 or Hq % cache.kv_heads:
            raise ValueError("the cache's kv_heads must divide the query heads")
        d.q_dev, d.q_stride[:] = _rows("q", rows, (cache.batch, n, Hq, cache.head_dim))
        d.q_heads, d.q_tokens, d.q_dtype = Hq, n, _DTYPES[q.dtype]
        if out is None:
            if out_dtype not in _DTYPES:
                raise ValueError("out_dtype must be fp32, bf16 or fp16")
            out = torch.empty(q.shape, dtype=out_dtype, device=q.device)
        if out.shape != q.shape or out.dtype not in _DTYPES or not out.is_contiguous():
            raise ValueError("out must be contiguous fp32/bf16/fp16 with the shape of q")
        d.out_dtype, d.out_dev = _DTYPES[out.dtype], out.data_ptr()
        d.causal, d.accumulate, d.split_tokens, d.scale = int(causal), int(accumulate), split_tokens, scale
        d.seq_lens_dev = _int32("lens", lens, (B,))
        d.q_lens_dev = _int32("q_lens", q_lens, (B,))
        self.lse = torch.empty(rows.shape[:3], dtype=torch.float32, device=q.device) if lse else None
        d.lse_dev = None if self.lse is None else self.lse.data_ptr()
        if weights is not None:
            if weights.dtype != torch.float32 or weights.dim() != 3 or tuple(weights.shape[:2]) != (B, cache.kv_heads) or \
                    weights.shape[2] < cache.max_tokens or not weights.is_contiguous():
                raise ValueError("weights must be contiguous fp32 [B, H, >= max_tokens]")
            d.weights_dev, d.weights_stride = weights.data_ptr(), weights.shape[2]
        size = L.lib().akv_q8_attention_workspace(ct.byref(d))
        if size == 0:
            L.check(L.lib().akv_q8_attention(ct.byref(d), None), "q8_attention")  # the status that says why
        self.workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
        d.workspace_dev, d.workspace_bytes = self.workspace.data_ptr(), size
        self.out, self.weights, self.cache = out, weights, cache
        self._prepare(d, cache.device, q, out, lens, q_lens, weights, self.lse, self.workspace, *_cache_tensors(cache))

    def run(self, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        self._issue(stream)
        return self.out


class Q8Evict(_Call):
    """Keep min(len, keep) tokens per sequence and kv head: the first `sinks`,
    the last `recent`, and those with the largest `weights` [B, H, T], packed
    in their order into `dst`, a cache in other memory (or in pages of the same
    pool that `src` has not got) that holds whole blocks.
    run() returns (kept token indices [B, H, keep] with -1 after the last,
    lengths [B], the kept tokens' weights [B, H, dst.max_tokens], 0 after the
    last): what the next steps go on with, in this object's own tensors, which
    its next run() writes anew."""

    _fn = "evict"

    def __init__(self, src: Q8Cache, dst: Q8Cache, weights: torch.Tensor, lens: torch.Tensor | None = None, *, keep: int,
                 sinks: int = 0, recent: int = 0):
        _on(src.device, dst=dst.k, weights=weights, lens=lens)
        if (src.fmt, src.batch, src.kv_heads, src.head_dim) != (dst.fmt, dst.batch, dst.kv_heads, dst.head_dim):
            raise ValueError("src and dst must agree in format, batch, kv_heads and head_dim")
        if not 0 < keep <= dst.max_tokens or sinks < 0 or recent < 0 or sinks + recent > keep:
            raise ValueError("keep must fit dst, and sinks + recent must fit keep")
        if dst.k.shape[2] % dst.block_tokens:
            raise ValueError("dst must hold whole blocks")
        B, H = src.batch, src.kv_heads
        if weights.dtype != torch.float32 or weights.dim() != 3 or tuple(weights.shape[:2]) != (B, H) or \
                weights.shape[2] < src.max_tokens or not weights.is_contiguous():
            raise ValueError("weights must be contiguous fp32 [B, H, >= max_tokens]")
        # Two block tables may share a pool: which pages they give out is on the device.
        one_pool = src.block_table is not None and dst.block_table is not None and src.block_table.data_ptr() != dst.block_table.data_ptr()
        if not one_pool and any(_may_overlap(a, b) for a in _planes(src) for b in _planes(dst)):
            raise ValueError("dst must not share memory with src")
        d = L.AkvQ8EvictDesc()
        d.src, d.dst = src._c, dst._c
        d.weights_dev, d.weights_stride = weights.data_ptr(), weights.shape[2]
        d.seq_lens_dev = _int32("lens", lens, (B,))
        d.keep, d.sinks, d.recent = keep, sinks, recent
        i32 = dict(dtype=torch.int32, device=src.device)
        self.kept = torch.empty(B, H, keep, **i32)
        self.lens = torch.empty(B, **i32)
        self.weights = torch.empty(B, H, dst.max_tokens, dtype=torch.float32, device=src.device)
        d.kept_dev, d.out_lens_dev = self.kept.data_ptr(), self.lens.data_ptr()
        d.out_weights_dev, d.out_weights_stride = self.weights.data_ptr(), dst.max_tokens
        d.out_weights_tokens = dst.max_tokens
        self.cache = dst
        self._prepare(d, src.device, weights, lens, self.kept, self.lens, self.weights, *_cache_tensors(src), *_cache_tensors(dst))

    def run(self, stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        self._issue(stream)
        return self.kept, self.lens, self.weights


def _capturing(stream: torch.cuda.Stream) -> bool:
    with torch.cuda.stream(stream):
        return torch.cuda.is_current_stream_capturing()


def _planes(c: Q8Cache) -> tuple:
    return c.k, c.v, c.k_scales, c.v_scales


def _cache_tensors(c: Q8Cache) -> tuple:
    return *_planes(c), c.block_table, c.status


def _may_overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors may have bytes in common. Views of different strides count as
    overlapping when the ranges do that they span; of equal strides, when an element of both
    can be at one place."""
    def span(t):
        return (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()
    if a.numel() == 0 or b.numel() == 0:
        return False
    apart = b.data_ptr() - a.data_ptr()
    if apart >= span(a) or -apart >= span(b):
        return False
    size = a.element_size()
    if a.stride() != b.stride() or size != b.element_size() or apart % size:
        return True
    dims = sorted(((s, n, m) for s, n, m in zip(a.stride(), a.shape, b.shape) if s and n * m > 1), reverse=True)

    def meet(left: int, dims: list) -> bool:
        # Is left = sum of s * (i - j) with 0 <= i < n, 0 <= j < m?
        if not dims:
            return left == 0
        s, n, m = dims[0]
        up, down = sum(r * (x - 1) for r, x, _ in dims[1:]), sum(r * (y - 1) for r, _, y in dims[1:])
        first, last = max(-(-(left - up) // s), 1 - m), min((left + down) // s, n - 1)
        return any(meet(left - s * k, dims[1:]) for k in range(first, last + 1))
    return meet(apart // size, dims)


def q8_store(cache: Q8Cache, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, counts: torch.Tensor | None = None,
             stream: torch.cuda.Stream | None = None) -> Q8Cache:
    """One `Q8Store`."""
    return Q8Store(cache, k, v, start, counts).run(stream)


def q8_restore(cache: Q8Cache, start: torch.Tensor | None, count: int, dtype: torch.dtype = torch.float32,
               stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """One `Q8Restore`."""
    return Q8Restore(cache, start, count, dtype).run(stream)


def q8_attention(q: torch.Tensor, cache: Q8Cache, lens: torch.Tensor | None = None, *, stream: torch.cuda.Stream | None = None,
                 **kw) -> torch.Tensor:
    """One `Q8Attention`."""
    return Q8Attention(q, cache, lens, **kw).run(stream)


def q8_evict(src: Q8Cache, dst: Q8Cache, weights: torch.Tensor, lens: torch.Tensor | None = None, *,
             stream: torch.cuda.Stream | None = None, **kw) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """One `Q8Evict`."""
    return Q8Evict(src, dst, weights, lens, **kw).run(stream)
