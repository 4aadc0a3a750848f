"""The operators of the 8-bit KV cache, as measured: storing tokens, attention
(with the attention weight each cached token received), eviction, restore.

A cache holds K and V as int8 or e4m3 codes with one fp32 scale for each block
of `block` tokens of a head: value = code * scale. Formulas, for one sequence
of `len` cached tokens whose newest `n` tokens are the queries:

  store    scale = amax / M over the block's new rows (M = 127, or 448 for
           e4m3), code = round(x / scale). A block that already holds rows
           keeps its scale unless the new rows need a larger one; its rows
           are then rounded again under the larger scale.
  attend   s[i, t] = scale * q[i] . K[t] for t <= len - n + i, p = softmax(s),
           out = p V; weights[h, t] += sum over the queries of kv head h's
           query heads of p (the accumulated attention weight of a token).
  evict    per kv head: the first `sinks` and the last `recent` tokens stay,
           the rest of `keep` goes to the tokens of the largest accumulated
           weight (ties: the lower index); the kept rows are packed, in order,
           into a new cache whose blocks get scales of their own.
  restore  code * scale, rounded once to the asked type.

A case is a dict: "op" and sizes. Lengths follow from the case alone, values
from the seed.
"""
import os
import random
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
MOST = {"int8": 127.0, "fp8": 448.0}


def listed():
    small = dict(batch=1, q_heads=9, kv_heads=3, dim=64)
    mid = dict(q_heads=32, kv_heads=8, dim=128)
    return [
        # One decode step of the smallest configuration: latency is all there is.
        dict(name="step 9/3 heads, 384", op="attend", tokens=384, q_tokens=1, ragged=False, page=0, fmt="int8", block=32,
             q_type="bf16", out_type="f32", weights=False, **small),
        # The default benchmark's shape: a batch of long sequences, one token each.
        dict(name="step B32, 32768", op="attend", batch=32, tokens=32768, q_tokens=1, ragged=False, page=0, fmt="int8",
             block=64, q_type="bf16", out_type="f32", weights=False, **mid),
        # Ragged sequences in shuffled 256-token pages, counting the weights that an eviction will need.
        dict(name="step ragged pages, weights", op="attend", batch=16, tokens=65536, q_tokens=1, ragged=True, page=256,
             fmt="fp8", block=32, q_type="bf16", out_type="f32", weights=True, **mid),
        # Few very long sequences of a 64/8-head layer: work has to be split along the tokens.
        dict(name="step B2, 131071, weights", op="attend", batch=2, q_heads=64, kv_heads=8, dim=128, tokens=131071, q_tokens=1,
             ragged=False, page=0, fmt="fp8", block=128, q_type="f16", out_type="f32", weights=True),
        # Five drafted tokens checked at once over ragged pages.
        dict(name="check 5 tokens, B8, 8192", op="attend", batch=8, tokens=8192, q_tokens=5, ragged=True, page=256, fmt="int8",
             block=64, q_type="f16", out_type="f16", weights=False, **mid),
        # A chunk of a long prompt against everything cached before it.
        dict(name="chunk 2048 of 32768", op="attend", batch=1, tokens=32768, q_tokens=2048, ragged=False, page=0, fmt="int8",
             block=64, q_type="bf16", out_type="bf16", weights=False, **mid),
        # A batch whose sequences bring chunks of odd lengths, with the weights.
        dict(name="chunks to 509, weights", op="attend", batch=4, q_heads=9, kv_heads=3, dim=64, tokens=8190, q_tokens=509,
             ragged=True, page=256, fmt="fp8", block=32, q_type="bf16", out_type="bf16", weights=True),
        # Every sequence of a batch appends its newest token to a block begun before.
        dict(name="store 1 token, B64", op="store", batch=64, kv_heads=8, dim=128, tokens=4096, new=1, ragged=True, page=256,
             fmt="fp8", block=32, q_type="bf16"),
        # Whole prompts, read in place from a projection that holds q, k and v side by side.
        dict(name="store 8192 tokens, B4", op="store", batch=4, kv_heads=8, dim=128, tokens=8192, new=8192, ragged=False, page=0,
             fmt="int8", block=64, q_type="bf16"),
        # One short-head layer reduced to an odd budget.
        dict(name="evict 8192 to 1001", op="evict", batch=1, kv_heads=3, dim=64, tokens=8192, keep=1001, sinks=4, recent=128,
             ragged=False, page=0, fmt="int8", block=32, q_type="bf16"),
        # A batch of long sequences in pages reduced to an eighth.
        dict(name="evict 32768 to 4096, B32", op="evict", batch=32, kv_heads=8, dim=128, tokens=32768, keep=4096, sinks=16,
             recent=512, ragged=True, page=256, fmt="fp8", block=64, q_type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    heads = rng.choice([(9, 3, 64), (32, 8, 128), (64, 8, 128), (16, 16, 64), (8, 1, 256), (12, 4, 96), (20, 5, 80)])
    c = dict(op=rng.choice(["attend", "attend", "attend", "store", "evict"]), batch=_log(rng, 1, 64), kv_heads=heads[1], dim=heads[2],
             tokens=_log(rng, 17, 131072), ragged=rng.random() < 0.6, page=rng.choice([0, 256]), fmt=rng.choice(["int8", "fp8"]),
             block=rng.choice([16, 32, 64, 128]), q_type=rng.choice(["bf16", "f16", "f32"]))
    if c["op"] == "attend":
        c["q_heads"] = heads[0]
        c["q_tokens"] = 1 if rng.random() < 0.5 else _log(rng, 2, min(2048, c["tokens"]))
        c["out_type"] = c["q_type"] if c["q_tokens"] > 1 or rng.random() < 0.5 else "f32"
        c["weights"] = rng.random() < 0.4
        # No more cache, scores or products than the listed cases have.
        while c["batch"] > 1 and (c["batch"] * c["kv_heads"] * c["tokens"] * c["dim"] > 1 << 30 or
                                  c["batch"] * heads[0] * c["q_tokens"] * c["tokens"] * c["dim"] > 1 << 38):
            c["batch"] -= 1
        while c["q_tokens"] > 1 and heads[0] * c["q_tokens"] * c["tokens"] * c["dim"] > 1 << 38:
            c["q_tokens"] -= 1
    else:
        if c["op"] == "store":
            c["new"] = 1 if rng.random() < 0.3 else _log(rng, 2, 8192)
            c["tokens"] = max(c["tokens"], c["new"] + 1)
            rows = max(c["new"], c["tokens"] // 8)
        else:
            c["keep"] = max(1, int(c["tokens"] * rng.uniform(0.05, 0.9)))
            c["sinks"] = min(c["keep"] // 4, rng.choice([0, 1, 4, 16]))
            c["recent"] = min(c["keep"] // 4, rng.choice([0, 1, 64, 512]))
            rows = max(c["keep"], c["tokens"] // 8)
        while c["batch"] > 1 and c["batch"] * c["kv_heads"] * rows * c["dim"] > 1 << 27:
            c["batch"] -= 1
    return c


def _lengths(case):
    """(cached tokens, new or query tokens) of each sequence: the case's own, odd ones among ragged ones."""
    b, t = case["batch"], case["tokens"]
    n = case.get("q_tokens", case.get("new", 1))
    if not case["ragged"]:
        return [t] * b, [n] * b
    r = random.Random("%d %d %d" % (b, t, n))
    lens, news = [], []
    for i in range(b):
        m = n if i == 0 else max(1, n - r.randrange(0, n // 2 + 1))
        lens.append(t if i == 0 else max(m, min(t, _log(r, max(1, t // 64), t) | 1)))
        news.append(m)
    return lens, news


def _starts(case):
    """Where each sequence's new tokens go."""
    lens, news = _lengths(case)
    return [max(0, n - m) for n, m in zip(lens, news)], news


def _window(case):
    """Rows of the whole blocks that new tokens can touch."""
    b = case["block"]
    return -(-(case["new"] + b - 1) // b) * b


def _capacity(case):
    """Tokens that the cache has room for: whole blocks, and room for every window."""
    b = case["page"] or case["block"]
    t = case["tokens"] + (_window(case) if case["op"] == "store" else 0)
    return -(-t // b) * b


def work(case):
    d, h, e = case["dim"], case["kv_heads"], {"f32": 4, "bf16": 2, "f16": 2}[case["q_type"]]
    lens, news = _lengths(case)
    if case["op"] == "attend":
        hq, cached, rows = case["q_heads"], sum(lens), case["batch"] * case["q_tokens"]
        pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lens, news))
        bytes_ = 2 * cached * h * (d + 4 / case["block"]) + rows * hq * d * (e + {"f32": 4, "bf16": 2, "f16": 2}[case["out_type"]])
        return {"bytes": bytes_ + (8 * cached * h if case["weights"] else 0), "flops": 4 * pairs * hq * d}
    if case["op"] == "store":
        new, window = sum(news), case["batch"] * _window(case)
        # Rows in, codes out, then the touched blocks read again and written as the values they stand for.
        return {"bytes": 2 * h * d * (new * (e + 1) + window * (1 + e)), "flops": 2 * h * d * (3 * new + window)}
    kept, seen = sum(min(n, case["keep"]) for n in lens), sum(lens)
    # Weights in, the kept rows in and out, then read again and written as the values they stand for.
    return {"bytes": h * (4 * seen + kept * (8 + 2 * d * (3 + e))), "flops": 2 * h * d * 5 * kept}


# ------------------------------------------------------------------- inputs

def _round8(y, fmt):
    """Codes, as floats, of values already divided by their scale."""
    m = MOST[fmt]
    y = y.clamp(-m, m)
    return y.round() if fmt == "int8" else y.to(torch.float8_e4m3fn).float()


def _scales(amax, fmt):
    return amax * (1.0 / MOST[fmt])


def _inverse(scale):
    """1 / scale, and 0 for a block of zeros."""
    return torch.where(scale > 0, scale.reciprocal(), torch.zeros_like(scale))


def _quantise(x, fmt):
    """x [..., rows of one block, dim] -> codes as floats, scale [...]."""
    s = _scales(x.abs().amax((-1, -2)), fmt)
    return _round8(x * _inverse(s)[..., None, None], fmt), s


def _values(shape, channel, g):
    """Values as keys and values of a layer: normal, each channel with a spread of its own."""
    return torch.randn(shape, generator=g, device=DEV) * channel


def _channels(h, d, g, outliers):
    c = torch.exp(0.5 * torch.randn(h, 1, d, generator=g, device=DEV))
    if outliers:
        at = torch.rand(h, 1, d, generator=g, device=DEV).argsort(-1)[..., :2]
        c.scatter_(-1, at, c.gather(-1, at) * 8)
    return c


def _cache(case, g):
    """K and V pools [pages, kv heads, page tokens, dim] with scales, and the
    table of each sequence's pages; a cache in one piece is one page a sequence."""
    b, h, d, blk, fmt = case["batch"], case["kv_heads"], case["dim"], case["block"], case["fmt"]
    cap = _capacity(case)
    page = case["page"] or cap
    per = cap // page
    pages = b * per
    s = {"block": blk, "page": page, "paged": bool(case["page"]), "cap": cap}
    for side in ("k", "v"):
        ch = _channels(h, d, g, side == "k")
        codes = torch.empty(pages, h, page, d, dtype=CODES[fmt], device=DEV)
        scales = torch.empty(pages, h, page // blk, device=DEV)
        step = max(1, (1 << 26) // (h * page * d))
        for i in range(0, pages, step):
            n = min(step, pages - i)
            x = _values((n, h, page, d), ch, g).view(n, h, page // blk, blk, d)
            c, sc = _quantise(x, fmt)
            codes[i:i + n] = c.view(n, h, page, d).to(CODES[fmt])
            scales[i:i + n] = sc
        s[side], s[side + "s"] = codes, scales
    order = torch.randperm(pages, generator=g, device=DEV) if case["page"] else torch.arange(pages, device=DEV)
    s["table"] = order.view(b, per).to(torch.int32)
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    b, h, d = case["batch"], case["kv_heads"], case["dim"]
    dt = TYPES[case["q_type"]]
    lens, news = _lengths(case)
    i32 = dict(dtype=torch.int32, device=DEV)
    s = _cache(case, g)
    s["case"] = case
    s["lens"] = torch.tensor(lens, **i32)
    if case["op"] == "attend":
        s["q"] = torch.randn(b, case["q_tokens"], case["q_heads"], d, generator=g, device=DEV).to(dt)
        s["news"] = torch.tensor(news, **i32)
        if case["weights"]:
            s["w"] = torch.rand(b, h, s["cap"], generator=g, device=DEV) * 4
    elif case["op"] == "store":
        starts, news = _starts(case)
        s["start"], s["news"] = torch.tensor(starts, **i32), torch.tensor(news, **i32)
        s["first"] = torch.tensor([t // case["block"] * case["block"] for t in starts], **i32)
        # Rows that nothing was stored in yet are zero.
        empty = torch.arange(s["cap"], device=DEV).view(1, -1) >= s["start"].view(-1, 1)
        mask = torch.empty_like(empty).view(-1, s["page"])
        mask[s["table"].view(-1).long()] = empty.view(-1, s["page"])
        for side in ("k", "v"):
            s[side].view(torch.int8).masked_fill_(mask[:, None, :, None], 0)
        # The new rows as a projection leaves them: q, k and v of a token side by side.
        n = case["new"]
        qkv = torch.randn(b, n, 3 * h, d, generator=g, device=DEV)
        qkv[:, :, h:2 * h] *= _channels(h, d, g, True).view(1, 1, h, d)
        qkv[:, :, 2 * h:] *= _channels(h, d, g, False).view(1, 1, h, d)
        qkv = qkv.to(dt)
        s["k_new"], s["v_new"] = qkv[:, :, h:2 * h], qkv[:, :, 2 * h:]
    else:
        # Accumulated weights: heavy-tailed, and nothing at all for some tokens.
        w = torch.exp(2 * torch.randn(b, h, s["cap"], generator=g, device=DEV) - 6)
        s["w"] = torch.where(torch.rand(b, h, s["cap"], generator=g, device=DEV) < 0.3, torch.zeros_like(w), w)
    if own:
        s["calls"] = _calls(s)
    return s


# ------------------------------------------------------ the framework's calls

def _calls(s):
    """The prepared calls that a serving program keeps for a layer."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "astc-kv_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import astc_kv_cuda as akv
    case = s["case"]
    table = dict(block_table=s["table"]) if s["paged"] else {}
    cache = akv.Q8Cache(s["k"], s["v"], s["ks"], s["vs"], block_tokens=s["block"], **table)
    dt = TYPES[case["q_type"]]
    if case["op"] == "attend":
        return [akv.Q8Attention(s["q"], cache, s["lens"], q_lens=s["news"], out_dtype=TYPES[case["out_type"]], weights=s.get("w"),
                                accumulate=True)]
    if case["op"] == "store":
        return [akv.Q8Store(cache, s["k_new"], s["v_new"], s["start"], counts=s["news"]),
                akv.Q8Restore(cache, s["first"], _window(case), dtype=dt)]
    to = akv.Q8Cache.zeros(case["batch"], case["kv_heads"], case["keep"], case["dim"], fmt=case["fmt"], block_tokens=case["block"])
    return [akv.Q8Evict(cache, to, s["w"], s["lens"], keep=case["keep"], sinks=case["sinks"], recent=case["recent"]),
            akv.Q8Restore(to, None, case["keep"], dtype=dt)]


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"attend": _attend, "store": _store, "evict": _evict}[op](s)
    calls = s["calls"]
    if op == "attend":
        out = calls[0].run()
        return [out, s["w"]] if s["case"]["weights"] else [out]
    if op == "store":
        calls[0].run()
        return list(calls[1].run())
    kept, lens, w = calls[0].run()
    return [kept, lens, w, *calls[1].run()]


# ------------------------------------------------------------ the plain forms

def _sequences(s, side):
    """Codes [batch, kv heads, capacity, dim] and scales [batch, kv heads, blocks] of every sequence."""
    c, sc = s[side], s[side + "s"]
    if not s["paged"]:
        return c, sc
    t = s["table"].long()
    b, per = t.shape
    c, sc = c.view(torch.int8)[t].view(c.dtype), sc[t]  # [b, per, h, ...]
    h, page, d = c.shape[2:]
    return c.transpose(1, 2).reshape(b, h, per * page, d), sc.transpose(1, 2).reshape(b, h, -1)


def _dequantised(s, side):
    c, sc = _sequences(s, side)
    b, h, t, d = c.shape
    return (c.float().view(b, h, -1, s["block"], d) * sc[..., None, None]).view(b, h, t, d)


def _attend(s):
    case = s["case"]
    b, h, d, n = case["batch"], case["kv_heads"], case["dim"], case["q_tokens"]
    g = case["q_heads"] // h
    k = _dequantised(s, "k")
    t = k.shape[2]
    q = s["q"].float().view(b, n, h, g, d).permute(0, 2, 3, 1, 4).reshape(b, h, g * n, d)
    sc = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5).view(b, h, g, n, t)
    del k
    i = torch.arange(n, device=DEV)
    lens, news = s["lens"].view(b, 1), s["news"].view(b, 1)
    ends = torch.where(i < news, lens - news + i + 1, torch.zeros_like(lens))  # [b, n]: tokens that a query sees
    seen = torch.arange(t, device=DEV) < ends[..., None]  # [b, n, t]
    sc.masked_fill_(~seen.view(b, 1, 1, n, t), float("-inf"))
    top = sc.amax(-1, keepdim=True)
    p = sc.sub_(torch.where(top > float("-inf"), top, torch.zeros_like(top))).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    out = torch.matmul(p.view(b, h, g * n, t), _dequantised(s, "v")).view(b, h, g, n, d)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, n, h * g, d).to(TYPES[case["out_type"]])
    if not case["weights"]:
        return [out]
    s["w"] += p.sum((2, 3))
    return [out, s["w"]]


def _store(s):
    case = s["case"]
    b, h, d, blk, fmt = case["batch"], case["kv_heads"], case["dim"], case["block"], case["fmt"]
    w = _window(case)
    j = torch.arange(w, device=DEV).view(1, w)
    off = (s["start"] - s["first"]).view(b, 1)
    at = s["first"].view(b, 1) + j  # [b, w] positions
    new = (j >= off) & (j < off + s["news"].view(b, 1))
    pages = s["table"].long().gather(1, (at // s["page"]).long())
    inside = (at % s["page"]).long()
    src = (j - off).clamp(0, case["new"] - 1).long()
    back = []
    for side in ("k", "v"):
        old = s[side].view(torch.int8)[pages, :, inside].view(s[side].dtype).float()  # [b, w, h, d]
        where = (pages[:, ::blk], slice(None), inside[:, ::blk] // blk)
        had = s[side + "s"][where]  # [b, w / blk, h]
        x = s[side + "_new"].gather(1, src[..., None, None].expand(b, w, h, d)).float()
        x = torch.where(new[..., None, None], x, torch.zeros_like(x)).view(b, -1, blk, h, d)
        need = _scales(x.abs().amax((2, 4)), fmt)
        begun = (at[:, ::blk] < s["start"].view(b, 1))[..., None]
        fresh = new.view(b, -1, blk).any(-1)[..., None]
        sc = torch.where(fresh, torch.where(begun, torch.maximum(had, need), need), had)
        inv = _inverse(sc)[:, :, None, :, None]
        old = old.view(b, -1, blk, h, d)
        again = _round8(old * had[:, :, None, :, None] * inv, fmt)
        moved = (begun & (sc > had))[:, :, None, :, None] & (at < s["start"].view(b, 1)).view(b, -1, blk, 1, 1)
        c = torch.where(new.view(b, -1, blk, 1, 1), _round8(x * inv, fmt), torch.where(moved, again, old))
        s[side].view(torch.int8)[pages, :, inside] = c.view(b, w, h, d).to(s[side].dtype).view(torch.int8)
        s[side + "s"][where] = sc
        back.append((c * sc[:, :, None, :, None]).view(b, w, h, d).to(TYPES[case["q_type"]]))
    return back


def _chosen(s):
    """Indices of the kept tokens [batch, kv heads, keep], ascending, -1 after the last; how many each sequence keeps."""
    case = s["case"]
    b, keep = case["batch"], case["keep"]
    t = torch.arange(s["cap"], device=DEV)
    lens = s["lens"].view(b, 1, 1)
    fixed = (t < case["sinks"]) | (t >= lens - case["recent"])
    w = torch.where(t < lens, torch.where(fixed, torch.full_like(s["w"], float("inf")), s["w"]), torch.full_like(s["w"], float("-inf")))
    best = w.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    n = s["lens"].clamp(max=keep)
    there = torch.arange(keep, device=DEV) < n.view(b, 1, 1)
    best = torch.where(there, best, torch.full_like(best, s["cap"])).sort(-1).values
    return torch.where(there, best, torch.full_like(best, -1)).to(torch.int32), n


def _evict(s):
    case = s["case"]
    b, h, d, blk, fmt, keep = case["batch"], case["kv_heads"], case["dim"], case["block"], case["fmt"], case["keep"]
    kept, n = _chosen(s)
    there = kept >= 0
    at = kept.clamp(min=0).long()
    w = torch.where(there, s["w"].gather(2, at), torch.zeros((), device=DEV))
    pages = s["table"].long().gather(1, (at // s["page"]).view(b, -1)).view(b, h, keep)
    inside, heads = at % s["page"], torch.arange(h, device=DEV).view(1, h, 1)
    rows = -(-keep // blk) * blk
    back = []
    for side in ("k", "v"):
        c = s[side].view(torch.int8)[pages, heads, inside].view(s[side].dtype).float()  # [b, h, keep, d]
        x = c * s[side + "s"][pages, heads, inside // blk][..., None]
        x = torch.where(there[..., None], x, torch.zeros_like(x))
        x = torch.cat([x, x.new_zeros(b, h, rows - keep, d)], 2).view(b, h, -1, blk, d)
        c, sc = _quantise(x, fmt)
        x = (c * sc[..., None, None]).view(b, h, rows, d)[:, :, :keep]
        back.append(x.transpose(1, 2).to(TYPES[case["q_type"]]).contiguous())
    return [kept, n, w, *back]


# ------------------------------------------------- the definitions in 64 bits

def _round8_exact(y, fmt):
    """The nearest code to y (ties to the even one), from what the formats are."""
    if fmt == "int8":
        return y.round().clamp(-127, 127)
    exponent = torch.frexp(y.abs().clamp(min=2.0 ** -9))[1] - 1  # |y| = 1.xxx * 2 ** exponent
    step = torch.exp2((exponent.clamp(min=-6) - 3).double())  # three bits after the leading one
    return (torch.round(y / step) * step).clamp(-448, 448)


def _row_values(s, side, b, h, at):
    """Values [tokens, dim] of the tokens `at` of one sequence and head, and their scales and codes."""
    pages, inside = s["table"][b].long()[at // s["page"]], at % s["page"]
    codes = s[side].view(torch.int8)[pages, h, inside].view(s[side].dtype).double()
    scales = s[side + "s"][pages, h, inside // s["block"]].double()
    return codes * scales[:, None], scales, codes


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _attend_exact, "store": _store_exact, "evict": _evict_exact}[case["op"]](s, case)


def _attend_exact(s, case):
    h, d = case["kv_heads"], case["dim"]
    g = case["q_heads"] // h
    lens, news = _lengths(case)
    out = torch.zeros(case["batch"], case["q_tokens"], case["q_heads"], d, dtype=torch.float64, device=DEV)
    w = s["w"].double() if case["weights"] else None
    for b, (n, m) in enumerate(zip(lens, news)):
        at = torch.arange(n, device=DEV)
        hidden = at[None] > torch.arange(n - m, n, device=DEV)[:, None]
        for j in range(h):
            k, v = _row_values(s, "k", b, j, at)[0], _row_values(s, "v", b, j, at)[0]
            for i in range(j * g, j * g + g):
                a = (s["q"][b, :m, i].double() @ k.T) / d ** 0.5
                p = torch.softmax(a.masked_fill(hidden, float("-inf")), 1)
                out[b, :m, i] = p @ v
                if w is not None:
                    w[b, j, :n] += p.sum(0)
    return [out] if w is None else [out, w]


def _store_exact(s, case):
    h, d, blk, w = case["kv_heads"], case["dim"], case["block"], _window(case)
    starts, news = _starts(case)
    back = []
    for side in ("k", "v"):
        all_ = torch.zeros(case["batch"], w, h, d, dtype=torch.float64, device=DEV)
        for b, (start, n) in enumerate(zip(starts, news)):
            first = start // blk * blk
            o = start - first
            x = torch.zeros(w, h, d, dtype=torch.float64, device=DEV)
            x[o:o + n] = s[side + "_new"][b, :n].double()
            x = x.view(-1, blk, h, d)
            sc = x.abs().amax((1, 3)) / MOST[case["fmt"]]
            if o:
                old = [_row_values(s, side, b, j, torch.arange(first, start, device=DEV)) for j in range(h)]
                had = torch.stack([v[1][0] for v in old])
                grown = torch.maximum(sc[0], had)
                for j, (values, _, _) in enumerate(old):
                    x[0, :o, j] = values if grown[j] == had[j] else _round8_exact(values / grown[j], case["fmt"]) * grown[j]
                sc[0] = grown
            f = sc[:, None, :, None].clamp(min=1e-300)
            y = _round8_exact(x / f, case["fmt"]) * f
            if o:  # the rows that were there are as above
                y[0, :o] = x[0, :o]
            all_[b] = y.view(w, h, d)
        back.append(all_)
    return back


def _evict_exact(s, case):
    h, d, blk, keep = case["kv_heads"], case["dim"], case["block"], case["keep"]
    lens, _ = _lengths(case)
    back = [torch.zeros(case["batch"], keep, h, d, dtype=torch.float64, device=DEV) for _ in "kv"]
    w = torch.zeros(case["batch"], h, keep, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        m = min(n, keep)
        a, z = min(case["sinks"], m), min(case["recent"], m)
        for j in range(h):
            if n <= keep:
                at = torch.arange(n, device=DEV)
            else:
                middle = s["w"][b, j, a:n - z].double()
                best = torch.sort(-middle, stable=True)[1][:keep - a - z] + a
                at = torch.cat([torch.arange(a, device=DEV), best.sort()[0], torch.arange(n - z, n, device=DEV)])
            w[b, j, :m] = s["w"][b, j, at].double()
            for side, to in zip("kv", back):
                x = torch.zeros(-(-keep // blk) * blk, d, dtype=torch.float64, device=DEV)
                x[:m] = _row_values(s, side, b, j, at)[0]
                x = x.view(-1, blk, d)
                f = (x.abs().amax((1, 2)) / MOST[case["fmt"]]).clamp(min=1e-300)[:, None, None]
                to[b, :, j] = (_round8_exact(x / f, case["fmt"]) * f).view(-1, d)[:keep]
    return [None, None, w, *back]
