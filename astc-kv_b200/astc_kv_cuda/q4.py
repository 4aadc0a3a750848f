"""The 4-bit KV cache: append with the position rotation on the way, attention,
restore on the GPU.

A `Q4Cache` holds K and V as e2m1 codes, two a byte, with an fp16 scale for
every 32 channels of a token (value = code * scale, rounded to fp16), in one
piece or in pages found through a block table: 4.5 bits a value. The calls
follow `Q8Attention`: an object that checks its tensors, builds the C
descriptor and its workspace once and is re-issued with `run()`, and a function
for a single call.

* `Q4Append` rotates the keys of new tokens, quantises keys and values into the
  cache and rotates the queries of the same tokens,
* `Q4Attention` attends one or many new tokens per sequence to it,
* `Q4Restore` returns tokens as values.

Lengths, positions and block tables are int32 CUDA tensors that are read when
a call runs, so a program updates them in place between steps. A call's
outputs and workspace are its own and written anew by every run: runs of one
call follow one another, on one stream or on streams that the program orders.
Everything below runs in libakv_cuda.so (C ABI: include/akv_q4.h, which has
the formulas and the rules for empty rows and values that are not finite).
"""
from __future__ import annotations

import ctypes as ct
from dataclasses import dataclass

import torch

from . import _lib as L
from .q8 import _DTYPES, _Call, _int32, _may_overlap, _on, _rows
from .rotary import Rotary

_GROUP, _TOKENS = L.AKV_Q4_GROUP, L.AKV_Q4_TOKENS


@dataclass(eq=False)
class Q4Cache:
    """K and V codes with their scales.

    One piece: codes uint8 [B, H, T, D / 2], scales fp16 [B, H, D / 32, T], T a
    multiple of 16. Paged: codes [num_pages, H, page_tokens, D / 2], scales
    [num_pages, H, D / 32, page_tokens], page_tokens a multiple of 16, and
    `block_table` int32 [B, pages_per_seq]. The lower channel of a byte is in
    its lower half. Codes and scales may be views whose last dimension is
    contiguous and whose other strides are multiples of 16 bytes (codes) or 4
    elements (scales). Sequences may share pages that they only read; what two
    appends write to one place is either one's. `max_tokens` (default: all there is
    room for) bounds a sequence. `status`: optional int32 [1] that kernels write an error code to
    (a bad table entry, tokens past the end, a position outside the rotary
    table, a wait inside a kernel that ran out); without it such rows are
    dropped, NaN or read as zeros and nothing says so.
    """
    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor
    block_table: torch.Tensor | None = None
    max_tokens: int = 0
    status: torch.Tensor | None = None

    def __post_init__(self):
        if self.k.dim() != 4 or self.k.dtype != torch.uint8:
            raise ValueError("codes must be uint8 [pages or B, H, tokens, D / 2]")
        if not self.k.is_cuda:
            raise ValueError("expected CUDA tensors")
        if self.v.shape != self.k.shape or self.v.dtype != self.k.dtype:
            raise ValueError("K and V codes must have the same shape and dtype")
        n, h, rows, half = self.k.shape
        d = 2 * half
        if d % _GROUP or not _GROUP <= d <= 256:
            raise ValueError("head_dim must be a multiple of 32, at most 256")
        if h < 1 or rows < 1 or rows % _TOKENS:
            raise ValueError("a cache needs heads, and tokens or pages in multiples of 16")
        for name in ("k", "v"):
            codes, scales = getattr(self, name), getattr(self, name + "_scales")
            if codes.stride(-1) != 1 or any(s % 16 for s in codes.stride()[:-1]) or codes.data_ptr() % 16:
                raise ValueError("codes need a contiguous last dimension, other strides in multiples of 16 bytes and 16-byte alignment")
            if scales.dtype != torch.float16 or tuple(scales.shape) != (n, h, d // _GROUP, rows) or scales.stride(-1) != 1 or \
                    any(s % 4 for s in scales.stride()[:-1]) or scales.data_ptr() % 8:
                raise ValueError(f"scales must be fp16 {[n, h, d // _GROUP, rows]} with a contiguous last dimension, "
                                 "other strides in multiples of 4 and 8-byte alignment")
        _on(self.device, v=self.v, k_scales=self.k_scales, v_scales=self.v_scales, block_table=self.block_table, status=self.status)
        if self.status is not None and (self.status.dtype != torch.int32 or self.status.numel() < 1):
            raise ValueError("status must be int32")
        if self.block_table is None:
            self.batch, room = n, rows
        else:
            if self.block_table.dim() != 2:
                raise ValueError("block_table must be [B, pages_per_seq]")
            _int32("block_table", self.block_table, tuple(self.block_table.shape))
            self.batch, room = self.block_table.shape[0], self.block_table.shape[1] * rows
        self.max_tokens = self.max_tokens or room
        if not 0 < self.max_tokens <= room:
            raise ValueError("max_tokens exceeds what the cache has room for")
        c = L.AkvQ4Cache()
        c.batch, c.kv_heads, c.head_dim = self.batch, h, d
        c.max_tokens, c.page_tokens = self.max_tokens, rows
        if self.block_table is not None:
            c.block_table_dev = self.block_table.data_ptr()
            c.pages_per_seq, c.num_pages = self.block_table.shape[1], n
        for name in ("k", "v"):
            codes, scales, side = getattr(self, name), getattr(self, name + "_scales"), L.AkvQ4Side()
            side.codes, side.scales, side.stride_token, side.scale_stride_group = codes.data_ptr(), scales.data_ptr(), codes.stride(2), scales.stride(2)
            side.stride_head, side.scale_stride_head = codes.stride(1), scales.stride(1)
            if self.block_table is None:
                side.stride_batch, side.scale_stride_batch = codes.stride(0), scales.stride(0)
            else:
                side.stride_page, side.scale_stride_page = codes.stride(0), scales.stride(0)
            setattr(c, name, side)
        c.status_dev = None if self.status is None else self.status.data_ptr()
        self._c = c

    @classmethod
    def zeros(cls, batch: int, kv_heads: int, max_tokens: int, head_dim: int, *, page_tokens: int = 0,
              block_table: torch.Tensor | None = None, num_pages: int = 0, status: torch.Tensor | None = None,
              device: torch.device | str = "cuda") -> "Q4Cache":
        """An empty cache: in one piece, or `num_pages` pages of `page_tokens` for a block table."""
        if block_table is None:
            n, rows = batch, -(-max_tokens // _TOKENS) * _TOKENS
        else:
            n, rows = num_pages, page_tokens

        def codes():
            return torch.zeros(n, kv_heads, rows, head_dim // 2, dtype=torch.uint8, device=device)

        def scales():
            return torch.zeros(n, kv_heads, head_dim // _GROUP, rows, dtype=torch.float16, device=device)
        return cls(codes(), codes(), scales(), scales(), block_table=block_table, max_tokens=max_tokens, status=status)

    @property
    def device(self) -> torch.device:
        return self.k.device

    @property
    def kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def head_dim(self) -> int:
        return 2 * self.k.shape[3]

    @property
    def nbytes(self) -> int:
        """Resident bytes: codes and scales."""
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scales, self.v_scales))


def _cache_tensors(c: Q4Cache) -> tuple:
    return c.k, c.v, c.k_scales, c.v_scales, c.block_table, c.status


class Q4Append(_Call):
    """Quantise k, v [B, n, H, D] into tokens start[b] .. start[b] + counts[b] - 1
    (n each without counts) of `cache`. With `rotary`, k is rotated first, at
    `positions` int32 [B, n] or [axes, B, n], or at the tokens' own places in the
    cache without positions; and `q` [B, n, Hq, D], the queries of the same tokens,
    is rotated to this object's own `q` (zeros past counts). Rows may be strided
    views, for example slices of a fused projection. run() returns the rotated
    queries, or the cache where there are none."""

    _family, _fn = "q4_", "append"

    def __init__(self, cache: Q4Cache, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, counts: torch.Tensor | None = None, *,
                 rotary: Rotary | None = None, positions: torch.Tensor | None = None, q: torch.Tensor | None = None):
        if k.dim() != 4:
            raise ValueError("k must be [B, n, H, D]")
        _on(cache.device, k=k, v=v, start=start, counts=counts, positions=positions, q=q, table=None if rotary is None else rotary.table)
        if start is None or k.dtype != v.dtype or (q is not None and q.dtype != k.dtype):
            raise ValueError("start is needed, and k, v and q must have one dtype")
        if rotary is None and (positions is not None or q is not None):
            raise ValueError("positions and q need a rotary table")
        if rotary is not None and 2 * rotary.pairs > cache.head_dim:
            raise ValueError("heads need as many channels as the pairs have")
        B, n = cache.batch, k.shape[1]
        d = L.AkvQ4AppendDesc()
        d.cache, d.tokens = cache._c, n
        shape = (B, n, cache.kv_heads, cache.head_dim)
        d.k_dev, d.k_stride[:] = _rows("k", k, shape)
        d.v_dev, d.v_stride[:] = _rows("v", v, shape)
        d.dtype = _DTYPES[k.dtype]
        d.start_dev = _int32("start", start, (B,))
        d.counts_dev = _int32("counts", counts, (B,))
        self.cache, self.q = cache, None
        if rotary is not None:
            d.rotary = rotary._c
            d.positions_dev = None if positions is None else rotary._places(positions, B, n)
        if q is not None:
            if q.dim() != 4 or q.shape[2] < 1:
                raise ValueError("q must be [B, n, Hq, D]")
            d.q_heads = q.shape[2]
            d.q_dev, d.q_stride[:] = _rows("q", q, (B, n, d.q_heads, cache.head_dim))
            self.q = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            d.q_out_dev = self.q.data_ptr()
        self._prepare(d, cache.device, k, v, start, counts, positions, q, self.q, None if rotary is None else rotary.table,
                      *_cache_tensors(cache))

    def run(self, stream: torch.cuda.Stream | None = None) -> torch.Tensor | Q4Cache:
        self._issue(stream)
        return self.cache if self.q is None else self.q


class Q4Restore(_Call):
    """Tokens start[b] + i (i without start), i < count, as values: (k, v) [B, count, H, D]."""

    _family, _fn = "q4_", "restore"

    def __init__(self, cache: Q4Cache, start: torch.Tensor | None, count: int, dtype: torch.dtype = torch.float16):
        if dtype not in _DTYPES:
            raise ValueError("dtype must be fp32, bf16 or fp16")
        if count < 0:
            raise ValueError("count must not be negative")
        _on(cache.device, start=start)
        shape = (cache.batch, count, cache.kv_heads, cache.head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=cache.device)
        self.v = torch.empty(shape, dtype=dtype, device=cache.device)
        d = L.AkvQ4RestoreDesc()
        d.cache, d.tokens, d.dtype = cache._c, count, _DTYPES[dtype]
        d.start_dev = _int32("start", start, (cache.batch,))
        d.k_dev, d.v_dev = self.k.data_ptr(), self.v.data_ptr()
        self._prepare(d, cache.device, self.k, self.v, start, *_cache_tensors(cache))

    def run(self, stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        self._issue(stream)
        return self.k, self.v


class Q4Attention(_Call):
    """Attention of the newest tokens of each sequence over the cache.

    q: [B, Hq, D] (one token per sequence) or [B, n, Hq, D], strided views
    allowed. `lens` int32 [B]: cached tokens per sequence, the queries' own
    included (None: the cache's max_tokens). `q_lens` int32 [B]: queries per
    sequence out of n (the rest of the output is zero). `causal`: query i sees
    tokens up to its own; otherwise every query sees the whole sequence.
    `out_dtype` fp32 (default) or a 16-bit type, which also lets the softmax
    weights meet V as fp16. Prompts want a 16-bit one: many rows (queries x
    heads of a kv head) of 16-bit queries and outputs go to another kernel, which
    takes 0.95 ms for 2048 tokens of 32768 (32/8 heads of 128 channels) where fp32
    outputs take 6.3. `lse=True` keeps ln sum exp of the scores in
    `self.lse` [B, n, Hq].

    Splits and workspace go by the cache's max_tokens, not by the lengths:
    where a cache has much more room than tokens, a second Q4Cache over the
    same tensors with a smaller `max_tokens` serves it faster (256 query tokens
    of 4096, 32/8 heads: room for 4096 39 us, for 131072 80).
    """

    _family, _fn = "q4_", "attention"

    def __init__(self, q: torch.Tensor, cache: Q4Cache, lens: torch.Tensor | None = None, *, q_lens: torch.Tensor | None = None,
                 causal: bool = True, scale: float = 0.0, out: torch.Tensor | None = None,
                 out_dtype: torch.dtype = torch.float32, lse: bool = False, split_tokens: int = 0):
        if q.dim() not in (3, 4):
            raise ValueError("q must be [B, Hq, D] or [B, n, Hq, D]")
        _on(cache.device, q=q, lens=lens, q_lens=q_lens, out=out)
        rows = q if q.dim() == 4 else q.unsqueeze(1)
        B, n, Hq, D = rows.shape
        d = L.AkvQ4AttnDesc()
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
        if _may_overlap(q, out):
            raise ValueError("out must not share memory with q")
        d.out_dtype, d.out_dev = _DTYPES[out.dtype], out.data_ptr()
        d.causal, d.split_tokens, d.scale = int(causal), split_tokens, scale
        d.seq_lens_dev = _int32("lens", lens, (B,))
        d.q_lens_dev = _int32("q_lens", q_lens, (B,))
        self.lse = torch.empty(rows.shape[:3], dtype=torch.float32, device=q.device) if lse else None
        d.lse_dev = None if self.lse is None else self.lse.data_ptr()
        size = L.lib().akv_q4_attention_workspace(ct.byref(d))
        if size == 0:
            L.check(L.lib().akv_q4_attention(ct.byref(d), None), "q4_attention")  # the status that says why
        self.workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
        d.workspace_dev, d.workspace_bytes = self.workspace.data_ptr(), size
        self.out, self.cache = out, cache
        self._prepare(d, cache.device, q, out, lens, q_lens, self.lse, self.workspace, *_cache_tensors(cache))

    def run(self, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        self._issue(stream)
        return self.out


def q4_append(cache: Q4Cache, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, counts: torch.Tensor | None = None, *,
              stream: torch.cuda.Stream | None = None, **kw) -> torch.Tensor | Q4Cache:
    """One `Q4Append`."""
    return Q4Append(cache, k, v, start, counts, **kw).run(stream)


def q4_restore(cache: Q4Cache, start: torch.Tensor | None, count: int, dtype: torch.dtype = torch.float16,
               stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """One `Q4Restore`."""
    return Q4Restore(cache, start, count, dtype).run(stream)


def q4_attention(q: torch.Tensor, cache: Q4Cache, lens: torch.Tensor | None = None, *, stream: torch.cuda.Stream | None = None,
                 **kw) -> torch.Tensor:
    """One `Q4Attention`."""
    return Q4Attention(q, cache, lens, **kw).run(stream)
