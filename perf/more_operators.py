"""The rotary positions and the 4-bit KV cache, as measured: rotating queries and
keys, appending tokens with the rotation on the way, attention.

  rotate   table[p][i] = cos, sin of p * theta^(-2i / R), in fp32. Pair i of a
           token takes the position of its axis (text has one axis, images
           height and width, video time, height and width). Pairs are channels
           (i, i + R/2), or (2i, 2i + 1) when interleaved; channels from R on
           stay. y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin; the inverse, which
           is the gradient, has -sin.
  append   K is rotated, K and V go into the cache: for each 32 channels of a
           token scale = fp16(amax / 6), code = the nearest e2m1 number (0, 0.5,
           1, 1.5, 2, 3, 4, 6; ties to the even code) to x / scale; queries of
           the same tokens are rotated. What a value in the cache stands for is
           code * scale, rounded to fp16.
  attend   s[i, t] = q[i] . K[t] / sqrt(D) for t <= len - n + i,
           out = softmax(s) V, for the newest n of `len` tokens.

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
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
GROUP = 32
THETA = 500000.0


def listed():
    small = dict(batch=1, q_heads=9, kv_heads=3, dim=64)
    mid = dict(q_heads=32, kv_heads=8, dim=128)
    one = dict(axes=1, interleaved=False)
    return [
        # One decode step of the smallest configuration: latency is all there is.
        dict(name="step 9/3 heads, 384", op="attend", tokens=384, q_tokens=1, ragged=False, page=0, q_type="bf16", out_type="f32", **small),
        # The default benchmark's shape: a batch of long sequences, one token each.
        dict(name="step B32, 32768", op="attend", batch=32, tokens=32768, q_tokens=1, ragged=False, page=0, q_type="bf16",
             out_type="bf16", **mid),
        # Ragged sequences in shuffled 256-token pages.
        dict(name="step ragged pages, 65536", op="attend", batch=16, tokens=65536, q_tokens=1, ragged=True, page=256, q_type="f16",
             out_type="f32", **mid),
        # Five drafted tokens checked at once over ragged pages, eight query heads a kv head.
        dict(name="check 5 tokens, B8, 8192", op="attend", batch=8, q_heads=64, kv_heads=8, dim=128, tokens=8192, q_tokens=5,
             ragged=True, page=256, q_type="f16", out_type="f16"),
        # A chunk of a long prompt against everything cached before it.
        dict(name="chunk 2048 of 32768", op="attend", batch=1, tokens=32768, q_tokens=2048, ragged=False, page=0, q_type="bf16",
             out_type="bf16", **mid),
        # A batch whose sequences bring chunks of odd lengths.
        dict(name="chunks to 509 of 8190", op="attend", batch=4, q_heads=9, kv_heads=3, dim=64, tokens=8190, q_tokens=509, ragged=True,
             page=256, q_type="bf16", out_type="bf16"),
        # A decode step's append: every sequence's newest token, queries rotated with it.
        dict(name="append 1 token, B64", op="append", batch=64, tokens=4096, new=1, ragged=True, page=256, rotary=128, queries=True,
             q_type="bf16", **one, **mid),
        # Whole prompts, read in place from a projection that holds q, k and v side by side.
        dict(name="append 8192 tokens, B4", op="append", batch=4, tokens=8192, new=8192, ragged=False, page=0, rotary=128, queries=True,
             q_type="bf16", **one, **mid),
        # A clip's tokens with time, height and width, odd counts, into pages.
        dict(name="append video, 1777 tokens", op="append", batch=2, q_heads=12, kv_heads=4, dim=96, tokens=8192, new=1777, ragged=True,
             page=256, rotary=96, queries=False, axes=3, interleaved=False, q_type="f16"),
        # One token's queries: latency.
        dict(name="rotate 1 token", op="rotate", batch=1, q_heads=32, dim=128, rotary=128, new=1, positions=131072, inverse=False,
             q_type="bf16", **one),
        # An image's patches, height and width, interleaved pairs, heads of an odd width.
        dict(name="rotate image, 4097 patches", op="rotate", batch=2, q_heads=16, dim=72, rotary=72, new=4097, positions=1024, axes=2,
             interleaved=True, inverse=False, q_type="f16"),
        # The gradient of long clips' queries and keys.
        dict(name="rotate video, gradient", op="rotate", batch=4, q_heads=40, dim=128, rotary=128, new=8191, positions=8192, axes=3,
             interleaved=False, inverse=True, q_type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "rotate"])
    c = dict(op=op, batch=_log(rng, 1, 64), q_type=rng.choice(["bf16", "f16", "f32"]))
    if op == "attend":
        c["q_heads"], c["kv_heads"], c["dim"] = rng.choice([(9, 3, 64), (32, 8, 128), (64, 8, 128), (16, 16, 64), (8, 1, 256), (12, 4, 96),
                                                            (20, 5, 160), (6, 2, 32)])
        c["tokens"], c["ragged"], c["page"] = _log(rng, 17, 131072), rng.random() < 0.6, rng.choice([0, 256])
        c["q_tokens"] = 1 if rng.random() < 0.5 else _log(rng, 2, min(2048, c["tokens"]))
        c["out_type"] = c["q_type"] if c["q_tokens"] > 1 or rng.random() < 0.5 else "f32"
        # No more cache, scores or products than the listed cases have.
        per = c["tokens"] * c["dim"]
        while c["batch"] > 1 and (c["batch"] * c["kv_heads"] * per > 1 << 30 or c["batch"] * c["q_heads"] * c["q_tokens"] * per > 1 << 38):
            c["batch"] -= 1
        while c["q_tokens"] > 1 and c["q_heads"] * c["q_tokens"] * per > 1 << 38:
            c["q_tokens"] -= 1
        return c
    c["axes"], c["interleaved"] = rng.choice([1, 1, 2, 3]), rng.random() < 0.3
    if op == "append":
        c["q_heads"], c["kv_heads"], c["dim"], c["rotary"] = rng.choice([(9, 3, 64, 64), (32, 8, 128, 128), (64, 8, 128, 64), (8, 1, 256, 128),
                                                                        (12, 4, 96, 96), (20, 5, 160, 160), (16, 16, 64, 32)])
        c["new"] = 1 if rng.random() < 0.3 else _log(rng, 2, 8192)
        c["tokens"], c["ragged"], c["page"] = max(_log(rng, 17, 32768), c["new"]), rng.random() < 0.6, rng.choice([0, 256])
        c["queries"] = rng.random() < 0.6
        while c["batch"] > 1 and c["batch"] * c["kv_heads"] * max(c["new"], c["tokens"] // 8) * c["dim"] > 1 << 25:
            c["batch"] -= 1
        return c
    c["q_heads"], c["dim"], c["rotary"] = rng.choice([(16, 64, 64), (16, 80, 80), (18, 72, 72), (40, 128, 128), (64, 128, 64), (12, 96, 48),
                                                      (8, 256, 128), (5, 160, 160), (1, 64, 64)])
    c["new"] = 1 if rng.random() < 0.2 else _log(rng, 2, 16384)
    c["positions"], c["inverse"] = max(c["new"], _log(rng, 1024, 131072)), rng.random() < 0.4
    while c["batch"] > 1 and c["batch"] * c["new"] * c["q_heads"] * c["dim"] > 1 << 27:
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


def _capacity(case):
    """Tokens that the cache has room for; an append reads a window of `new` tokens back."""
    unit = case["page"] or 16
    t = case["tokens"] + (case["new"] if case["op"] == "append" else 0)
    return -(-t // unit) * unit


def _axis_of(case):
    """The axis of each pair: the first of three gets a quarter of the pairs, the others share the rest."""
    pairs, a = case["rotary"] // 2, case["axes"]
    cuts = [0] if a == 1 else [0, pairs // 2] if a == 2 else [0, pairs // 4, pairs // 4 + (pairs - pairs // 4) // 2]
    return [sum(i >= c for c in cuts) - 1 for i in range(pairs)]


def work(case):
    d, e = case["dim"], SIZE[case["q_type"]]
    if case["op"] == "rotate":
        tokens = case["batch"] * case["new"]
        return {"bytes": 2 * tokens * case["q_heads"] * d * e + min(tokens, case["positions"]) * case["rotary"] * 4,
                "flops": 3 * tokens * case["q_heads"] * case["rotary"]}
    h, hq = case["kv_heads"], case["q_heads"]
    lens, news = _lengths(case)
    row = d / 2 + d / GROUP * 2  # of the cache
    if case["op"] == "attend":
        pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lens, news))
        rows = case["batch"] * case["q_tokens"] * hq * d
        return {"bytes": 2 * sum(lens) * h * row + rows * (e + SIZE[case["out_type"]]), "flops": 4 * pairs * hq * d}
    new, back, heads = sum(news), case["batch"] * case["new"], hq if case["queries"] else 0
    # Rows in, codes out, the window read again and written as the fp16 values it stands for, queries in and out.
    bytes_ = 2 * h * (new * (d * e + row) + back * (row + 2 * d)) + heads * d * e * (new + back) + min(new, max(lens)) * case["rotary"] * 4
    return {"bytes": bytes_, "flops": 2 * h * d * (5 * new + back) + 3 * new * heads * d}


# ------------------------------------------------------------------- inputs

def _channels(h, d, g, outliers):
    c = torch.exp(0.5 * torch.randn(h, 1, d, generator=g, device=DEV))
    if outliers:
        at = torch.rand(h, 1, d, generator=g, device=DEV).argsort(-1)[..., :2]
        c.scatter_(-1, at, c.gather(-1, at) * 8)
    return c


def _cache(case, g, empty):
    """K and V codes [pages, kv heads, page tokens, dim / 2] with scales [pages, kv heads, dim / 32, page tokens] and the table of
    each sequence's pages; a cache in one piece is one page a sequence."""
    b, h, d = case["batch"], case["kv_heads"], case["dim"]
    cap = _capacity(case)
    page = case["page"] or cap
    per = cap // page
    pages = b * per
    s = {"page": page, "paged": bool(case["page"]), "cap": cap}
    for side in ("k", "v"):
        codes = torch.zeros(pages, h, page, d // 2, dtype=torch.uint8, device=DEV)
        scales = torch.zeros(pages, h, d // GROUP, page, dtype=torch.float16, device=DEV)
        ch = _channels(h, d, g, side == "k")
        step = max(1, (1 << 26) // (h * page * d))
        for i in range(0, 0 if empty else pages, step):
            n = min(step, pages - i)
            codes[i:i + n], sc = _quantise(torch.randn(n, h, page, d, generator=g, device=DEV) * ch)
            scales[i:i + n] = sc.transpose(-1, -2)
        s[side], s[side + "s"] = codes, scales
    order = torch.randperm(pages, generator=g, device=DEV) if case["page"] else torch.arange(pages, device=DEV)
    s["table"] = order.view(b, per).to(torch.int32)
    return s


def _rotary_table(positions, rotary):
    inv = THETA ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=DEV) / rotary)
    a = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def _places(first, n, axes, most):
    """Positions [axes, batch, n] of n tokens from `first` [batch] on: in reading order, or of a picture or clip that begins there."""
    i = torch.arange(n, device=DEV).view(1, n)
    w = max(1, round((n / axes) ** (1 / axes))) if axes > 1 else 1
    at = [i] if axes == 1 else [i // w, i % w] if axes == 2 else [i // (w * w), i // w % w, i % w]
    return torch.stack([(first.view(-1, 1) + x).clamp(max=most - 1) for x in at]).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    b, d, dt, hq = case["batch"], case["dim"], TYPES[case["q_type"]], case["q_heads"]
    i32 = dict(dtype=torch.int32, device=DEV)
    if case["op"] == "rotate":
        n, most = case["new"], case["positions"]
        s = {"x": torch.randn(b, n, hq, d, generator=g, device=DEV).to(dt), "rotary": _rotary_table(most, case["rotary"])}
        first = torch.randint(0, max(1, most - n + 1), (b,), generator=g, device=DEV)
        s["places"] = _places(first, n, case["axes"], most)
    else:
        lens, news = _lengths(case)
        s = _cache(case, g, case["op"] == "append")
        s["lens"], s["news"] = torch.tensor(lens, **i32), torch.tensor(news, **i32)
        if case["op"] == "attend":
            s["q"] = torch.randn(b, case["q_tokens"], hq, d, generator=g, device=DEV).to(dt)
        else:
            # The new rows as a projection leaves them: q, k and v of a token side by side.
            n, h = case["new"], case["kv_heads"]
            qkv = torch.randn(b, n, hq + 2 * h, d, generator=g, device=DEV)
            qkv[:, :, hq:hq + h] *= _channels(h, d, g, True).view(1, 1, h, d)
            qkv[:, :, hq + h:] *= _channels(h, d, g, False).view(1, 1, h, d)
            qkv = qkv.to(dt)
            s["q"], s["k_new"], s["v_new"] = qkv[:, :, :hq], qkv[:, :, hq:hq + h], qkv[:, :, hq + h:]
            s["start"] = s["lens"] - s["news"]
            s["rotary"] = _rotary_table(s["cap"], case["rotary"])
            s["places"] = _places(s["start"], n, case["axes"], s["cap"])
    s["case"] = case
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
    if case["op"] != "attend":
        rotary = akv.Rotary(s["rotary"], axes=_axis_of(case), interleaved=case["interleaved"])
        if case["op"] == "rotate":
            return [akv.Rotate(s["x"], rotary, s["places"], inverse=case["inverse"])]
    table = dict(block_table=s["table"]) if s["paged"] else {}
    cache = akv.Q4Cache(s["k"], s["v"], s["ks"], s["vs"], **table)
    if case["op"] == "attend":
        return [akv.Q4Attention(s["q"], cache, s["lens"], q_lens=s["news"], out_dtype=TYPES[case["out_type"]])]
    return [akv.Q4Append(cache, s["k_new"], s["v_new"], s["start"], counts=s["news"], rotary=rotary, positions=s["places"],
                         q=s["q"] if case["queries"] else None),
            akv.Q4Restore(cache, s["start"], case["new"], dtype=torch.float16)]


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"attend": _attend, "append": _append, "rotate": _rotate}[op](s)
    if op != "append":
        return [s["calls"][0].run()]
    q = s["calls"][0].run()
    back = list(s["calls"][1].run())
    return back + [q] if s["case"]["queries"] else back


# ------------------------------------------------------------ the plain forms

def _quantise(x):
    """x [..., dim] -> codes [..., dim / 2] (two a byte, the lower channel in the lower half), scales [..., dim / 32]."""
    x = x.reshape(*x.shape[:-1], -1, GROUP)
    sc = (x.abs().amax(-1) / 6).half().clamp(max=10912)
    y = x / torch.where(sc > 0, sc.float(), torch.full_like(x[..., 0], float("inf")))[..., None]
    a = y.abs()
    c = (a > 0.25).to(torch.uint8)
    c += a >= 0.75
    c += a > 1.25
    c += a >= 1.75
    c += a > 2.5
    c += a >= 3.5
    c += a > 5
    c |= torch.signbit(y).to(torch.uint8) << 3
    c = c.reshape(*c.shape[:-2], -1, 2)
    return c[..., 0] | c[..., 1] << 4, sc


def _values(codes, scales):
    """Values, as fp32, of codes [..., dim / 2] with scales [..., dim / 32]."""
    number = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float16, device=DEV)
    number = torch.cat([number, -number])
    i = torch.arange(256, device=DEV)
    pair = torch.stack([number[i % 16], number[i // 16]], 1).view(torch.int32)[:, 0]
    x = pair.index_select(0, codes.reshape(-1).int()).view(torch.float16)
    x = x.view(*scales.shape, GROUP) * scales[..., None]
    return x.flatten(-2).float()


def _sequences(s, side):
    """Values [batch, kv heads, capacity, dim] of every sequence."""
    c, sc = s[side], s[side + "s"].transpose(-1, -2)
    if s["paged"]:
        t = s["table"].long()
        b, per = t.shape
        c, sc = c[t].transpose(1, 2), sc[t].transpose(1, 2)  # [b, h, per, page, ...]
        c, sc = c.reshape(b, c.shape[1], per * s["page"], -1), sc.reshape(b, sc.shape[1], per * s["page"], -1)
    return _values(c, sc)


def _attend(s):
    case = s["case"]
    b, h, d, n = case["batch"], case["kv_heads"], case["dim"], case["q_tokens"]
    g = case["q_heads"] // h
    k = _sequences(s, "k")
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
    out = torch.matmul(p.view(b, h, g * n, t), _sequences(s, "v")).view(b, h, g, n, d)
    return [out.permute(0, 3, 1, 2, 4).reshape(b, n, h * g, d).to(TYPES[case["out_type"]])]


def _turned(x, s, case):
    """x [batch, n, heads, dim] rotated, in fp32."""
    axis = torch.tensor(_axis_of(case), device=DEV)
    r, pairs = case["rotary"], case["rotary"] // 2
    at = s["places"].long()[axis]  # [pairs, batch, n]
    both = s["rotary"][at, torch.arange(pairs, device=DEV).view(-1, 1, 1)]  # [pairs, batch, n, 2]
    c, z = (both[..., i].permute(1, 2, 0)[:, :, None] for i in (0, 1))
    if case.get("inverse"):
        z = -z
    x = x.float()
    turn, rest = x[..., :r], x[..., r:]
    x1, x2 = (turn[..., 0::2], turn[..., 1::2]) if case["interleaved"] else (turn[..., :pairs], turn[..., pairs:])
    y1, y2 = x1 * c - x2 * z, x2 * c + x1 * z
    y = torch.stack([y1, y2], -1).flatten(-2) if case["interleaved"] else torch.cat([y1, y2], -1)
    return torch.cat([y, rest], -1)


def _rotate(s):
    return [_turned(s["x"], s, s["case"]).to(s["x"].dtype)]


def _append(s):
    case = s["case"]
    b, n = case["batch"], case["new"]
    i = torch.arange(n, device=DEV).view(1, n)
    new = i < s["news"].view(b, 1)
    at = (s["start"].view(b, 1) + i).long()
    pages, inside = s["table"].long().gather(1, at // s["page"]), at % s["page"]
    back = []
    for side, x in (("k", _turned(s["k_new"], s, case)), ("v", s["v_new"].float())):
        codes, sc = _quantise(x)
        here, over = (s[side], (pages, slice(None), inside)), (s[side + "s"], (pages, slice(None), slice(None), inside))
        here[0][here[1]] = codes = torch.where(new[..., None, None], codes, here[0][here[1]])
        over[0][over[1]] = sc = torch.where(new[..., None, None], sc, over[0][over[1]])
        back.append(_values(codes, sc).half())
    if case["queries"]:
        q = _turned(s["q"], s, case)
        back.append(torch.where(new[..., None, None], q, torch.zeros_like(q)).to(s["q"].dtype))
    return back


# ------------------------------------------------- the definitions in 64 bits

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _row_values(s, side, b, h, at):
    """Values [tokens, dim] of the tokens `at` of one sequence and head."""
    pages, inside = s["table"][b].long()[at // s["page"]], at % s["page"]
    byte = s[side][pages, h, inside].long()
    code = torch.stack([byte & 15, byte >> 4], -1).flatten(-2)
    x = torch.tensor(LEVELS, dtype=torch.float64, device=DEV)[code & 7] * (1 - 2 * (code >> 3)).double()
    sc = s[side + "s"][pages, h][torch.arange(len(at), device=DEV), :, inside].double().repeat_interleave(GROUP, -1)
    return (x * sc).half().double()


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _attend_exact, "append": _append_exact, "rotate": _rotate_exact}[case["op"]](s, case)


def _attend_exact(s, case):
    h, d = case["kv_heads"], case["dim"]
    g = case["q_heads"] // h
    lens, news = _lengths(case)
    out = torch.zeros(case["batch"], case["q_tokens"], case["q_heads"], d, dtype=torch.float64, device=DEV)
    for b, (n, m) in enumerate(zip(lens, news)):
        at = torch.arange(n, device=DEV)
        hidden = at[None] > torch.arange(n - m, n, device=DEV)[:, None]
        for j in range(h):
            k, v = _row_values(s, "k", b, j, at), _row_values(s, "v", b, j, at)
            for i in range(j * g, j * g + g):
                a = (s["q"][b, :m, i].double() @ k.T) / d ** 0.5
                out[b, :m, i] = torch.softmax(a.masked_fill(hidden, float("-inf")), 1) @ v
    return [out]


def _turned_exact(x, s, case):
    """As complex numbers, pair by pair: (x1 + i x2) e^(i angle)."""
    r = case["rotary"]
    y = x.double().clone()
    for i, a in enumerate(_axis_of(case)):
        angle = s["places"][a].double() * THETA ** (-2.0 * i / r) * (-1 if case.get("inverse") else 1)
        turn = torch.polar(torch.ones_like(angle), angle)[..., None]
        p, q = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
        z = torch.complex(y[..., p], y[..., q]) * turn
        y[..., p], y[..., q] = z.real, z.imag
    return y


def _rotate_exact(s, case):
    return [_turned_exact(s["x"], s, case)]


def _append_exact(s, case):
    n = case["new"]
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=DEV)
    middles = (levels[1:] + levels[:-1]) / 2
    there = torch.arange(n, device=DEV) < s["news"].view(-1, 1)
    back = []
    for x in (_turned_exact(s["k_new"], s, case), s["v_new"].double()):
        x = x.unflatten(-1, (-1, GROUP))
        sc = (x.abs().amax(-1, keepdim=True) / 6).half().double().clamp(max=10912)
        y = x / sc.clamp(min=2.0 ** -24)
        low = torch.bucketize(y.abs(), middles)  # a value in the middle gets the lower one,
        high = torch.bucketize(y.abs(), middles, right=True)  # here the higher one
        x = (levels[torch.where(low % 2 == 0, low, high)].copysign(y) * sc).half().double().flatten(-2)
        back.append(torch.where(there[..., None, None], x, torch.zeros_like(x)))
    if case["queries"]:
        q = _turned_exact(s["q"], s, case)
        back.append(torch.where(there[..., None, None], q, torch.zeros_like(q)))
    return back
