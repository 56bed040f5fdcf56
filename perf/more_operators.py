"""The work that the operators around a served paged cache are timed on: its block tables and slot maps, rotary
positions with several axes, bounds of its pages' keys, and attention over the pages that a query selects by them.

A case is a dict of plain values; `op` says which operator it goes through:

    "reserve"  paged_reserve: pages for the tokens that requests bring, with their slots and positions
    "rotary"   rotary of queries and keys by positions of several axes, alone or with its gradients
    "append"   paged_append: rotation by such positions, new rows into the pages, the pages' bounds kept
    "bounds"   paged_bounds: the least and the largest value of each channel over the keys of a page
    "select"   paged_select and sdpa_paged: the pages that could matter most to a query, and attention over them

Pages hold bf16 (`bits` 16) or 4 bits per value (`bits` 4). `listed()` gives the cases that stand for the
range, `draw()` more of the same ranges.

Pages of 4 bits: uint8 [pages, kv heads, page size, D / 2 + D / 16], of which each 16 tokens of a head are one
block: 16 D / 2 bytes of codes, then per token D / 64 words of 32 bits, one for each group of 64 channels, that
hold bf16 (step, least value) from the low bits up. A code c stands for least + step * c. The order of the codes
inside a block is _places().
"""

import functools
import math

import torch

own = False


def _ktt():
    import kohaku_tt_b200 as ktt

    return ktt


# ---- the ranges -------------------------------------------------------------------------

def _spread(rng, low, high):
    """A whole number from low to high, spread evenly over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


GROUPED = [(14, 2), (16, 2), (16, 4), (32, 8)]      # query heads, key / value heads
PLAIN = [(8, 8), (12, 12), (16, 16)]


def _reserve(batch, tokens, keys, page):
    """1 to `tokens` new ones of each sequence behind up to `keys` cached ones."""
    return {"op": "reserve", "batch": batch, "tokens": tokens, "keys": keys, "page": page}


def _rotary(batch, heads, kv_heads, tokens, dim, part, axes, spread, interleaved, grad, packed=False, dtype="bf16"):
    """`tokens` of each sequence, or of the packed batch; `part`: the columns that turn; `axes` of the positions, whose pairs
    lie in runs, or take turns (`spread`)."""
    return {"op": "rotary", "batch": batch, "heads": heads, "kv_heads": kv_heads, "tokens": tokens, "dim": dim, "part": part, "axes": axes,
            "spread": spread, "interleaved": interleaved, "grad": grad, "packed": packed, "dtype": dtype}


def _append(bits, batch, heads, kv_heads, tokens, keys, dim, part, axes, spread, page, packed=False):
    """`tokens` new ones of each sequence (packed: at most) behind up to `keys` cached ones."""
    return {"op": "append", "bits": bits, "batch": batch, "heads": heads, "kv_heads": kv_heads, "tokens": tokens, "keys": keys,
            "dim": dim, "part": part, "axes": axes, "spread": spread, "page": page, "packed": packed}


def _bounds(bits, batch, kv_heads, keys, dim, page):
    return {"op": "bounds", "bits": bits, "batch": batch, "kv_heads": kv_heads, "keys": keys, "dim": dim, "page": page}


def _select(bits, batch, heads, kv_heads, tokens, keys, dim, page, top, first, last, packed=False):
    """`tokens` queries of each sequence (packed: at most) over up to `keys` keys, these queries' own among them: each goes to `top`
    pages, the `first` and the `last` of its sequence among them."""
    return {"op": "select", "bits": bits, "batch": batch, "heads": heads, "kv_heads": kv_heads, "tokens": tokens, "keys": keys,
            "dim": dim, "page": page, "top": top, "first": first, "last": last, "packed": packed}


def _draw_reserve(rng):
    tokens = rng.choice([1, 1, _spread(rng, 2, 64), _spread(rng, 64, 4096)])
    return _reserve(_spread(rng, 1, max(1, min(512, 262144 // tokens))), tokens, _spread(rng, 16, 8192), rng.choice([16, 32, 64]))


def _draw_rotary(rng):
    h, hk = rng.choice(GROUPED + PLAIN)
    d = rng.choice([64, 80, 96, 128])
    part = rng.choice([d, d, d // 2, 2 * rng.randint(4, d // 2)])
    tokens = _spread(rng, 1, 65536)
    batch = _spread(rng, 1, max(1, min(64, 65536 // tokens)))
    packed = rng.random() < 0.4
    return _rotary(batch, h, hk, tokens, d, part, rng.choice([2, 3, 3]), rng.random() < 0.4, rng.random() < 0.3, rng.random() < 0.5, packed,
                   rng.choice(["bf16", "bf16", "fp16", "fp32"]))


def _draw_append(rng):
    h, hk = rng.choice(GROUPED + PLAIN)
    d = rng.choice([64, 128])
    packed = rng.random() < 0.6
    tokens = _spread(rng, 8, 2048) if packed else rng.choice([1, 1, 1, _spread(rng, 2, 256)])
    keys = _spread(rng, 64, 4096)
    batch = _spread(rng, 1, max(1, min(64, 8192 // tokens, 131072 // (tokens + keys))))
    return _append(rng.choice([16, 4]), batch, h, hk, tokens, keys, d, rng.choice([d, d, d // 2]), rng.choice([2, 3, 3]), rng.random() < 0.4,
                   rng.choice([16, 32, 64]), packed)


def _draw_bounds(rng):
    _, hk = rng.choice(GROUPED + PLAIN)
    keys = _spread(rng, 64, 16384)
    return _bounds(rng.choice([16, 4]), _spread(rng, 1, max(1, min(64, 65536 // keys))), hk, keys, rng.choice([64, 128]), rng.choice([16, 32, 64]))


def _draw_select(rng):
    h, hk = rng.choice(GROUPED + PLAIN)
    page = rng.choice([16, 32, 64])
    tokens = rng.choice([1, 1, 1, rng.randint(2, 16)])
    keys = max(_spread(rng, 512, 65536), 2 * tokens)
    batch = _spread(rng, 1, max(1, min(64, 2097152 // (keys * hk), 256 // tokens)))
    first = rng.choice([0, 1, 1, 4])
    last = rng.choice([1, 2, 8])
    top = first + last + _spread(rng, 1, 2048 // page)
    return _select(rng.choice([16, 4]), batch, h, hk, tokens, keys, rng.choice([64, 128]), page, top, first, last, tokens > 1 and rng.random() < 0.5)


FAMILIES = [
    # The tables of a server's step: one token of a full batch, of which every 16th sequence or so needs a page; and prompts
    # of many lengths that come in at once.
    ([dict(_reserve(64, 1, 4096, 16), name="reserve token"),
      dict(_reserve(128, 2048, 1024, 16), name="reserve prompts")], _draw_reserve),
    # A short prompt around a small picture before its attention; and a training step on packed sequences of text, pictures and
    # video: the largest pass.
    ([dict(_rotary(1, 14, 2, 77, 64, 64, 3, False, False, False), name="rotary axes short"),
      dict(_rotary(16, 16, 16, 65536, 128, 128, 3, True, False, True, packed=True), name="rotary axes train")], _draw_rotary),
    # The neighbours of a token of a full server batch whose pages have bounds; and prompts with pictures, some of them behind
    # what is cached already, into 4 bits, with the check that a server makes of it: the cache read back.
    ([dict(_append(16, 64, 16, 2, 1, 1024, 128, 128, 3, False, 16), name="append token, bounds"),
      dict(_append(4, 8, 32, 8, 2048, 2048, 128, 128, 3, False, 16, packed=True), name="append prompts, bounds")], _draw_append),
    # A cached prefix that gets its bounds: a short one in 4 bits, and a server's in bf16.
    ([dict(_bounds(4, 1, 2, 1024, 64, 16), name="bounds short, 4 bits"),
      dict(_bounds(16, 16, 8, 8192, 128, 32), name="bounds")], _draw_bounds),
    # Generating text behind long contexts by 1,024 or 2,048 of their keys: one sequence; a full server batch in bf16 and in 4 bits;
    # and a few drafted tokens each of several sequences, each with its own pages.
    ([dict(_select(16, 1, 32, 8, 1, 65536, 128, 64, 32, 1, 2), name="select one long"),
      dict(_select(16, 64, 16, 2, 1, 16384, 128, 16, 64, 1, 4), name="select batch"),
      dict(_select(4, 64, 16, 2, 1, 16384, 128, 16, 64, 1, 4), name="select batch, 4 bits"),
      dict(_select(16, 8, 14, 2, 5, 8192, 64, 16, 64, 1, 2, packed=True), name="select drafts")], _draw_select),
]


def listed():
    return [dict(case) for cases, _ in FAMILIES for case in cases]


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


@functools.lru_cache(None)
def _most():
    return max(_cost(case) for case in listed())


def draw(rng):
    family = rng.choice([_draw_reserve, _draw_reserve, _draw_rotary, _draw_rotary, _draw_append, _draw_append, _draw_bounds, _draw_select, _draw_select,
                         _draw_select])
    while True:
        case = family(rng)
        if _cost(case) <= _most():
            return case


# ---- the pages --------------------------------------------------------------------------

@functools.lru_cache(None)
def _places(dim, value):
    """[16 D]: which nibble of a block holds the code of (token, channel). Eight channels share a word of 32
    bits, channel e of them at nibble (e >> 1) + 4 (e & 1). Keys: a token's words lie together, the one of
    channels 32 i + 8 t .. at place t D / 32 + i. Values: two tokens' words of channels 8 g .. (and 64 + 8 g ..)
    lie together, at a place that changes from pair to pair."""
    token, channel = torch.arange(16)[:, None], torch.arange(dim)[None, :]
    e = channel % 8
    nibble = (e >> 1) + 4 * (e & 1)
    if value:
        pair, g, wide = token // 2, channel // 8 % 8, dim // 64
        place = g ^ (2 * (pair & 3) if dim == 128 else 4 * (pair >> 1 & 1))
        word = (pair * 8 + place) * 2 * wide + (token & 1) * wide + channel // 64
    else:
        word = token * (dim // 8) + channel // 8 % 4 * (dim // 32) + channel // 32
    return (word * 8 + nibble).reshape(-1).cuda()


def _quantise(x):
    """Codes, step and least value of fp32 values [..., D] by groups of 64 channels."""
    x = x.unflatten(-1, (-1, 64))
    least, most = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step = ((most - least) * (1.0 / 15)).to(torch.bfloat16).float()
    code = torch.where(step > 0, torch.round((x - least) / step), torch.zeros_like(x)).clamp(0, 15)
    return code.flatten(-2), step.squeeze(-1), least.squeeze(-1)


def _values(code, step, least):
    return (least.unsqueeze(-1) + step.unsqueeze(-1) * code.unflatten(-1, (-1, 64))).flatten(-2)


def _pack(x, value):
    """Values [pages, Hk, page, D] in 4 bits: uint8 [pages, Hk, page, D / 2 + D / 16]."""
    n, hk, page, d = x.shape
    code, step, least = _quantise(x.float())
    nibbles = torch.empty((n, hk, page // 16, 16 * d), dtype=torch.uint8, device=x.device)
    nibbles[..., _places(d, value)] = code.reshape(n, hk, page // 16, 16 * d).to(torch.uint8)
    codes = nibbles[..., 0::2] | nibbles[..., 1::2] << 4
    words = torch.stack([step, least], dim=-1).to(torch.bfloat16).view(torch.uint8).reshape(n, hk, page // 16, d)
    return torch.cat([codes, words], dim=-1).reshape(n, hk, page, d // 2 + d // 16)


def _parts_of(pages, value):
    """Codes, steps and least values [..., page, D or D / 64] of pages of 4 bits."""
    *lead, page, wide = pages.shape
    d = wide * 16 // 9
    blocks = pages.reshape(*lead, page // 16, 16 * wide)
    codes, words = blocks[..., :8 * d], blocks[..., 8 * d:].contiguous()
    nibbles = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    code = nibbles[..., _places(d, value)].reshape(*lead, page, d).float()
    pairs = words.view(torch.bfloat16).reshape(*lead, page, d // 64, 2).float()
    return code, pairs[..., 0], pairs[..., 1]


def _rows_in(pages, value):
    """fp32 values [..., page, D] of pages."""
    return _values(*_parts_of(pages, value)) if pages.dtype == torch.uint8 else pages.float()


def _bounds_of(pages, live):
    """(least, largest) of each channel over the keys `live` [..., page] of pages [..., Hk, page, D], bf16 [..., Hk, 2, D]; zeros
    where none is live."""
    x, live = _rows_in(pages, False), live[..., None, :, None]
    least = torch.where(live, x, torch.full_like(x, math.inf)).amin(-2)
    most = torch.where(live, x, torch.full_like(x, -math.inf)).amax(-2)
    out = torch.stack([least, most], dim=-2)
    return torch.where(live.any(-2, keepdim=True), out, torch.zeros_like(out)).to(torch.bfloat16)


# ---- inputs -----------------------------------------------------------------------------

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _lengths(case, seed):
    """What the sequences of a case have: the tokens of each (packed rotary; None: dense), the keys of each (bounds), or the new
    tokens of each and the keys that are cached (reserve, append: before them; select: in all), uniform over the range."""
    g = torch.Generator().manual_seed(seed)

    def of(low, high, n):
        return torch.randint(low, high + 1, (n,), generator=g).tolist()

    if case["op"] == "rotary":
        if not case["packed"]:
            return None
        each = max(1, case["tokens"] // case["batch"])
        cut = [min(case["tokens"], max(1, n)) for n in of(each // 2, each + each // 2, case["batch"] - 1)]
        while sum(cut) >= case["tokens"] and cut:
            cut.pop()
        return cut + [case["tokens"] - sum(cut)]
    b, n = case["batch"], case["keys"]
    cached = of(max(1, n // 8), n, b)
    if case["op"] == "bounds":
        return cached
    new = [case["tokens"]] * b
    if case.get("packed") or case["op"] == "reserve":   # each sequence with an opposite, so that all seeds have as many tokens
        low, high = max(1, case["tokens"] // 4), case["tokens"]
        new = of(low, high, b // 2)
        new += [low + high - n for n in new] + [(low + high) // 2] * (b % 2)
    if case["op"] == "select":
        cached = [max(x, y) for x, y in zip(cached, new)]
    elif case.get("packed") or case["tokens"] > 64:
        cached = [0 if i % 2 else x for i, x in enumerate(cached)]
    return new, cached


def _normal(g, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _tables(positions, part, base=10000.0):
    """The plan that a program keeps: fp32 cosines and sines."""
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * base ** (-torch.arange(0, part, 2, device="cuda", dtype=torch.float64) / part)
    return angle.cos().float(), angle.sin().float()


def _axes(case):
    """The axis of each pair of columns: runs of a quarter (time) and the rest in equal shares, or one after another in turn."""
    n, axes = case["part"] // 2, case["axes"]
    if case["spread"]:
        return tuple(i % axes for i in range(n))
    time = n // 4
    return tuple(0 if i < time else 1 + (i - time) * (axes - 1) // (n - time) for i in range(n))


def _places_of(case, n, start, seed):
    """[axes, n] positions of a sequence's n tokens from position `start`: runs of text, where all axes count on, and pictures, whose
    rows and columns (and frames, the first axis) count from the position they begin at."""
    g = torch.Generator().manual_seed(seed)
    axes, parts, have = case["axes"], [], 0
    at = start
    while have < n:
        text = int(torch.randint(1, 48, (1,), generator=g))
        parts.append((at + torch.arange(text)).expand(axes, text))
        at += text
        frames, high, wide = (int(x) for x in torch.randint(1, 24, (3,), generator=g))
        frames = 1 + frames // 16
        t, y, x = torch.meshgrid(torch.arange(frames), torch.arange(high), torch.arange(wide), indexing="ij")
        grid = torch.stack([t, y, x])[3 - axes:].reshape(axes, -1)
        parts.append(at + grid)
        at += max(frames, high, wide)
        have += text + grid.shape[1]
    return torch.cat(parts, dim=1)[:, :n]


def _cumulative(lengths):
    return torch.tensor([0] + lengths).cumsum(0).to(device="cuda", dtype=torch.int32)


def _wide(case):
    """Pages that a sequence may have."""
    return -(-(case["keys"] + (case["tokens"] if case["op"] in ("append", "reserve") else 0)) // case["page"])


def _named(g, case, rows):
    """A table that names pages in no order for the `rows` of each sequence, and none behind them; the pages; and those it leaves."""
    b, wide = case["batch"], _wide(case)
    names = torch.randperm(b * wide, generator=g, device="cuda").to(torch.int32)
    table = torch.full((b, wide), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(-(-n // case["page"]) for n in rows):
        table[i, :n] = names[at:at + n]
        at += n
    return table, b * wide, names[at:].contiguous()


def _pool(g, case, count, value):
    hk, d, page = case["kv_heads"], case["dim"], case["page"]
    if case["bits"] == 16:
        return _normal(g, count, hk, page, d)
    return torch.cat([_pack(_normal(g, min(2048, count - i), hk, page, d), value) for i in range(0, count, 2048)])


def _live(table, lengths, count, page):
    """[pages, page] which rows of the pages are keys of a sequence."""
    live = torch.zeros((count, page), dtype=torch.bool, device="cuda")
    row = torch.arange(table.shape[1] * page, device="cuda").view(1, -1, page) < lengths[:, None, None]
    there = table >= 0
    live[table[there].long()] = row.expand(table.shape[0], -1, -1)[there]
    return live


def _bounds_in_parts(k_pages, live):
    return torch.cat([_bounds_of(k_pages[i:i + 4096], live[i:i + 4096]) for i in range(0, k_pages.shape[0], 4096)])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    lengths = _lengths(case, seed)
    if case["op"] == "rotary":
        n, d, dtype = case["tokens"], case["dim"], DTYPES[case["dtype"]]
        if case["packed"]:
            at = torch.cat([_places_of(case, x, 0, seed + i) for i, x in enumerate(lengths)], dim=1)
            shapes = [(n, case["heads"], d), (n, case["kv_heads"], d)]
        else:
            at = torch.stack([_places_of(case, n, 0, seed + i) for i in range(case["batch"])], dim=1)
            shapes = [(case["batch"], case["heads"], n, d), (case["batch"], case["kv_heads"], n, d)]
        state["positions"] = at.to(device="cuda", dtype=torch.int32).contiguous()
        state["axes"] = _axes(case)
        state["cos"], state["sin"] = _tables(int(at.max()) + 1, case["part"])
        state["q"], state["k"] = (_normal(g, *s, dtype=dtype).requires_grad_(case["grad"]) for s in shapes)
        if case["grad"]:
            state["dq"], state["dk"] = (_normal(g, *s, dtype=dtype) for s in shapes)
        return state
    if case["op"] == "bounds":
        state["table"], count, _ = _named(g, case, lengths)
        state["k_pages"] = _pool(g, case, count, False)
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        state["bounds"] = torch.zeros((count, case["kv_heads"], 2, case["dim"]), dtype=torch.bfloat16, device="cuda")
        return state
    new, cached = lengths
    state["lengths"] = torch.tensor(cached, dtype=torch.int32, device="cuda")
    if case["op"] == "reserve":
        state["table"], count, free = _named(g, case, cached)
        state["free"] = torch.cat([free, free.new_full((count - free.numel(),), -1)])
        state["count"] = torch.tensor([free.numel()], dtype=torch.int32, device="cuda")
        state["added"], state["tokens"] = torch.tensor(new, dtype=torch.int32, device="cuda"), sum(new)
        state["next"] = torch.empty_like(state["count"])
        return state
    append, d = case["op"] == "append", case["dim"]
    state["table"], count, _ = _named(g, case, [x + y for x, y in zip(new, cached)] if append else cached)
    state["k_pages"], state["v_pages"] = _pool(g, case, count, False), _pool(g, case, count, True)
    state["bounds"] = _bounds_in_parts(state["k_pages"], _live(state["table"], state["lengths"], count, case["page"]))
    state["cu"] = _cumulative(new) if case["packed"] else None
    n, h, hk, b = sum(new), case["heads"], case["kv_heads"], case["batch"]
    state["q"] = _normal(g, n, h, d) if case["packed"] else _normal(g, b, h, case["tokens"], d)
    if append:
        shape = (n, hk, d) if case["packed"] else (b, hk, case["tokens"], d)
        state["k"], state["v"] = _normal(g, *shape), _normal(g, *shape)
        each = [_places_of(case, x, y, seed + i) for i, (x, y) in enumerate(zip(new, cached))]
        at = torch.cat(each, dim=1) if case["packed"] else torch.stack(each, dim=1)
        state["positions"] = at.to(device="cuda", dtype=torch.int32).contiguous()
        state["axes"] = _axes(case)
        state["cos"], state["sin"] = _tables(max(int(at.max()) + 1, state["table"].shape[1] * case["page"]), case["part"])
        state["next"] = torch.empty_like(state["lengths"])
    return state


# ---- one pass ---------------------------------------------------------------------------

def _plain_reserve(s):
    page, wide = s["case"]["page"], s["table"].shape[1]
    lengths, added, free, table = s["lengths"].long(), s["added"].long(), s["free"], s["table"]
    held, wanted = (lengths + page - 1) // page, (lengths + added + page - 1) // page
    taken = (wanted - held).cumsum(0)
    granted = (taken <= s["count"]).to(torch.int64).cumprod(0).bool()
    entry = torch.arange(wide, device="cuda")
    mine = (entry >= held[:, None]) & (entry < wanted[:, None])
    place = s["count"].long() - 1 - (taken - (wanted - held))[:, None] - (entry - held[:, None])     # from the end of the list on
    names = torch.where(granted[:, None], free[place.clamp(0, free.numel() - 1)], torch.full_like(table, -1))
    table.copy_(torch.where(mine, names, table))
    s["next"].copy_(s["count"] - (torch.where(granted, wanted - held, torch.zeros_like(held))).sum())
    cu = torch.cat([added.new_zeros(1), added.cumsum(0)]).to(torch.int32)
    row = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(cu[1:].contiguous(), row.to(torch.int32), right=True)
    at = lengths[seq] + row - cu.long()[seq]
    slots = torch.where(granted[seq], table[seq, at // page].long() * page + at % page, torch.full_like(at, -1))
    return {"cu": cu, "positions": at.to(torch.int32), "slots": slots, "granted": torch.where(granted, added, torch.zeros_like(added)).to(torch.int32),
            "table": table, "count": s["next"]}


def _angles(s):
    """cos, sin [..., R / 2] of each token by the positions' axes."""
    axis = torch.tensor(s["axes"], device="cuda")
    at, pair = s["positions"].long().movedim(0, -1)[..., axis], torch.arange(len(s["axes"]), device="cuda")
    return s["cos"][at, pair], s["sin"][at, pair]


def _turn(x, cos, sin, interleaved):
    """fp32 rotation of the first columns of x [..., D] by cos, sin [..., R / 2]; rounded to x's type."""
    r = 2 * cos.shape[-1]
    head, rest = x[..., :r].float(), x[..., r:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else head.chunk(2, dim=-1)
    y1, y2 = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([y1, y2], dim=-1).flatten(-2) if interleaved else torch.cat([y1, y2], dim=-1)
    return torch.cat([y.to(x.dtype), rest], dim=-1)


def _plain_rotary(s):
    case = s["case"]
    cos, sin = (x.unsqueeze(1) for x in _angles(s))     # (the heads: of [T, H, D], or of [B, H, S, D])
    q, k = (_turn(s[name].detach(), cos, sin, case["interleaved"]) for name in ("q", "k"))
    if not case["grad"]:
        return {"q": q, "k": k}
    dq, dk = (_turn(s[name], cos, -sin, case["interleaved"]) for name in ("dq", "dk"))   # the transposed rotation
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _rows_of(s, n):
    """Sequence and place in its new tokens of each of n token rows of a packed batch."""
    at = torch.arange(n, device="cuda")
    seq = torch.searchsorted(s["cu"][1:].contiguous(), at.to(torch.int32), right=True)
    return seq, at - s["cu"].long()[seq]


def _plain_bounds(s, bounds, since, lengths):
    """The bounds of the pages that keys since .. lengths - 1 lie in, from all of their keys."""
    page, table = s["case"]["page"], s["table"]
    entry = torch.arange(table.shape[1], device="cuda")
    seq, at = torch.nonzero((entry >= (since // page)[:, None]) & (entry * page < lengths[:, None]), as_tuple=True)
    for i in range(0, seq.numel(), 4096):
        b, e = seq[i:i + 4096], at[i:i + 4096]
        live = e[:, None] * page + torch.arange(page, device="cuda") < lengths[b][:, None]
        names = table[b, e].long()
        bounds[names] = _bounds_of(s["k_pages"][names], live)
    return bounds


def _plain_append(s):
    case, page = s["case"], s["case"]["page"]
    cos, sin = (x.unsqueeze(1) for x in _angles(s))
    if case["packed"]:
        seq, place = _rows_of(s, s["q"].shape[0])
        at = s["lengths"].long()[seq] + place
        k_rows, v_rows = _turn(s["k"], cos, sin, False), s["v"]
        added = s["cu"][1:] - s["cu"][:-1]
    else:
        b, n = case["batch"], case["tokens"]
        at = (s["lengths"].long()[:, None] + torch.arange(n, device="cuda")).flatten()
        k_rows, v_rows = (x.transpose(1, 2).flatten(0, 1) for x in (_turn(s["k"], cos, sin, False), s["v"]))
        seq, added = torch.arange(b, device="cuda").repeat_interleave(n), n
    to, row = s["table"][seq, at // page].long(), at % page
    s["next"].copy_(s["lengths"] + added)
    out = {"q": _turn(s["q"], cos, sin, False), "lengths": s["next"]}
    for name, rows, value in (("k", k_rows, False), ("v", v_rows, True)):
        pages = s[name + "_pages"]
        if case["bits"] == 16:
            pages[to, :, row] = rows
            out[name] = pages
            continue
        # Whole pages that the new rows lie in, taken apart and put together again.
        names, inside = torch.unique(to, return_inverse=True)
        dense = _rows_in(pages[names], value).to(torch.bfloat16)
        dense[inside, :, row] = rows
        fresh = torch.zeros((names.numel(), page), dtype=torch.bool, device="cuda")
        fresh[inside, row] = True
        packed = _pack(dense, value)
        pages[names] = _merged(pages[names], packed, fresh, value)
        wide = s["table"].shape[1] * page
        there = (torch.arange(wide, device="cuda") < s["next"][:, None])[:, None, :, None]
        got = _rows_in(pages[s["table"].clamp(min=0).long()], value).transpose(1, 2).flatten(2, 3)
        out[name] = torch.where(there, got, torch.zeros_like(got)).to(torch.bfloat16)
    out["bounds"] = _plain_bounds(s, s["bounds"], s["lengths"], s["next"])
    return out


def _merged(old, new, fresh, value):
    """Pages of 4 bits whose rows `fresh` [pages, page] are those of `new`."""
    n, hk, page, wide = old.shape
    d = wide * 16 // 9
    word = torch.empty(16 * d, dtype=torch.int64, device="cuda")
    word[_places(d, value)] = torch.arange(16, device="cuda").repeat_interleave(d)      # the token of each nibble
    token = torch.cat([word[0::2], torch.arange(16, device="cuda").repeat_interleave(d // 16)])   # of each byte of a block
    taken = fresh.view(n, 1, page // 16, 16)[..., token].reshape(n, 1, page, wide)
    return torch.where(taken, new, old)


def _tokens_of(s):
    """Of each query token of a "select" case: its sequence, and the keys it sees; the queries [T, H, D]."""
    case = s["case"]
    if case["packed"]:
        seq, place = _rows_of(s, s["q"].shape[0])
        added = (s["cu"][1:] - s["cu"][:-1]).long()[seq]
        return seq, s["lengths"].long()[seq] - added + place + 1, s["q"]
    b, n = case["batch"], case["tokens"]
    seq = torch.arange(b, device="cuda").repeat_interleave(n)
    place = torch.arange(n, device="cuda").repeat(b)
    return seq, s["lengths"].long()[seq] - n + place + 1, s["q"].transpose(1, 2).flatten(0, 1)


def _plain_select(s):
    case, page, top = s["case"], s["case"]["page"], s["case"]["top"]
    seq, seen, q = _tokens_of(s)
    t, h, d = q.shape
    hk, wide = case["kv_heads"], s["table"].shape[1]
    count = (seen + page - 1) // page
    # The largest logit that a key between a page's bounds could have, of the queries that share a head. In 64 bits: what is
    # chosen should not depend on an order of summation.
    scores = torch.empty((t, hk, wide), dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        mine = torch.nonzero(seq == b)[:, 0]
        bounds = s["bounds"][s["table"][b].clamp(min=0).long()].double()     # [wide, Hk, 2, D]
        x = q[mine].double().view(-1, hk, h // hk, d)
        least, most = bounds[:, :, 0].permute(1, 2, 0), bounds[:, :, 1].permute(1, 2, 0)
        scores[mine] = (x.clamp(min=0) @ most + x.clamp(max=0) @ least).amax(2)
    entry = torch.arange(wide, device="cuda")
    there = (entry < count[:, None])[:, None]
    kept = ((entry < case["first"]) | (entry >= (count - case["last"])[:, None]))[:, None]
    scores = torch.where(kept, torch.full_like(scores, math.inf), scores)
    scores = torch.where(there, scores, torch.full_like(scores, -math.inf))
    order = torch.sort(scores, dim=-1, descending=True, stable=True).indices[..., :top]
    order = torch.nn.functional.pad(order, (0, top - order.shape[-1]), value=wide)
    order = torch.where(order < count[:, None, None], order, torch.full_like(order, wide)).sort(dim=-1).values
    names = torch.nn.functional.pad(s["table"], (0, 1), value=-1)[seq[:, None, None], order]
    many = count.clamp(max=top)
    keys = ((many - 1) * page + (seen - 1) % page + 1).to(torch.int32)[:, None].expand(t, hk).contiguous()

    rows = [names.clamp(min=0).long(), torch.arange(hk, device="cuda")[None, :, None]]
    k, v = (_rows_in(s[name][rows[0], rows[1]], value).flatten(2, 3) for name, value in (("k_pages", False), ("v_pages", True)))
    logits = (q.float().view(t, hk, h // hk, d) @ k.transpose(-1, -2)) / math.sqrt(d)
    live = (torch.arange(top * page, device="cuda") < keys[..., None])[:, :, None]
    logits = torch.where(live, logits, torch.full_like(logits, -math.inf))
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    out = ((p / p.sum(-1, keepdim=True)) @ v).reshape(t, h, d)
    if not case["packed"]:
        out = out.view(case["batch"], case["tokens"], h, d).transpose(1, 2)
    return {"chosen": names, "keys": keys, "out": out.to(torch.bfloat16)}


def run(s):
    case = s["case"]
    if not own:
        with torch.no_grad():
            if case["op"] == "bounds":
                return _plain_bounds(s, s["bounds"], torch.zeros_like(s["lengths"]), s["lengths"])
            return {"reserve": _plain_reserve, "rotary": _plain_rotary, "append": _plain_append, "select": _plain_select}[case["op"]](s)
    ktt = _ktt()
    if case["op"] == "reserve":
        cu, positions, slots, granted = ktt.paged_reserve(s["table"], s["lengths"], s["added"], s["free"], s["count"], case["page"], s["tokens"],
                                                          count_out=s["next"])
        return {"cu": cu, "positions": positions, "slots": slots, "granted": granted, "table": s["table"], "count": s["next"]}
    if case["op"] == "rotary":
        q, k = ktt.rotary(s["q"], s["k"], s["cos"], s["sin"], positions=s["positions"], interleaved=case["interleaved"], axes=s["axes"])
        if not case["grad"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if case["op"] == "append":
        q = ktt.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], cos=s["cos"], sin=s["sin"], q=s["q"],
                             cu_seq=s["cu"], lengths_out=s["next"], positions=s["positions"], axes=s["axes"], bounds=s["bounds"])
        if case["bits"] == 16:
            return {"q": q, "lengths": s["next"], "k": s["k_pages"], "v": s["v_pages"], "bounds": s["bounds"]}
        k, v = ktt.paged_read(s["k_pages"], s["v_pages"], s["table"], s["next"])
        return {"q": q, "lengths": s["next"], "k": k, "v": v, "bounds": s["bounds"]}
    if case["op"] == "bounds":
        return ktt.paged_bounds(s["k_pages"], s["table"], s["lengths"], bounds=s["bounds"])
    chosen, keys = ktt.paged_select(s["q"], s["bounds"], s["table"], s["lengths"], case["page"], case["top"], first=case["first"], last=case["last"],
                                    cu_seq_q=s["cu"])
    return {"chosen": chosen, "keys": keys, "out": ktt.sdpa_paged(s["q"], s["k_pages"], s["v_pages"], chosen, keys)}


# ---- the definition in 64 bits ----------------------------------------------------------

def _exact_turn(x, s, at, inverse=False):
    """x [n, H, D] turned at positions `at` [axes, n], pair by pair as complex numbers; nothing rounded."""
    x, n = x.double(), len(s["axes"])
    y = x.clone()
    for i, axis in enumerate(s["axes"]):
        first, second = (2 * i, 2 * i + 1) if s["case"].get("interleaved") else (i, i + n)
        row = at[axis].long()
        turn = torch.complex(s["cos"][row, i].double(), s["sin"][row, i].double() * (-1 if inverse else 1))[:, None]
        z = torch.complex(x[..., first], x[..., second]) * turn
        y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rows(s, name, i, n):
    """Row-major [n, heads, D] of sequence i."""
    if s["cu"] is None:
        return s[name][i].transpose(0, 1)
    at = int(s["cu"][i])
    return s[name][at:at + n]


def _exact_pages(pages, value):
    """[..., page, D] in 64 bits."""
    if pages.dtype != torch.uint8:
        return pages.double()
    code, step, least = (x.double() for x in _parts_of(pages, value))
    return least.repeat_interleave(64, -1) + step.repeat_interleave(64, -1) * code


def _exact_sequence(pages, table, n, value):
    """The first n rows of a sequence, [n, Hk, D] in 64 bits, from its pages."""
    return _exact_pages(pages[table[:-(-n // pages.shape[2])].long()], value).transpose(1, 2).flatten(0, 1)[:n]


def _exact_four_bits(x):
    """What a row [n, Hk, D] of bf16 values is worth once it is held in 4 bits."""
    x = x.to(torch.bfloat16).double().unflatten(-1, (-1, 64))
    least, most = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step = ((most - least) / 15).to(torch.bfloat16).double()
    return (least + step * torch.round((x - least) / step.clamp(min=1e-300)).clamp(0, 15)).flatten(-2)


def _exact_bounds(rows, page):
    """[pages, Hk, 2, D] of the keys [n, Hk, D] of a sequence."""
    return torch.stack([torch.stack([x.amin(0), x.amax(0)], dim=1) for x in rows.split(page)])


def _exact_reserve(s, new, cached):
    page, table, free, left = s["case"]["page"], s["table"].tolist(), s["free"].tolist(), int(s["count"])
    cu, positions, slots, granted, short = [0], [], [], [], False
    for row, n, have in zip(table, new, cached):
        held, wanted = -(-have // page), -(-(have + n) // page)
        short = short or wanted - held > left
        for e in range(held, wanted):
            row[e] = -1
            if not short:
                left -= 1
                row[e] = free[left]
        cu.append(cu[-1] + n)
        positions += range(have, have + n)
        slots += [-1 if short else row[j // page] * page + j % page for j in range(have, have + n)]
        granted.append(0 if short else n)

    def of(x, dtype=torch.int32):
        return torch.tensor(x, dtype=dtype, device="cuda")

    return {"cu": of(cu), "positions": of(positions), "slots": of(slots, torch.int64), "granted": of(granted), "table": of(table), "count": of([left])}


def exact(case, seed):
    s = prepare(case, seed)
    lengths = _lengths(case, seed)
    if case["op"] == "reserve":
        return _exact_reserve(s, *lengths)
    if case["op"] == "rotary":
        out = {}
        for name in ("q", "k", "dq", "dk") if case["grad"] else ("q", "k"):
            x, back = s[name].detach(), name[0] == "d"
            if case["packed"]:
                out[name] = _exact_turn(x, s, s["positions"], back)
            else:
                out[name] = torch.stack([_exact_turn(y.transpose(0, 1), s, s["positions"][:, i], back).transpose(0, 1) for i, y in enumerate(x)])
        return out
    if case["op"] == "bounds":
        out = s["bounds"].double()
        for i, n in enumerate(lengths):
            names = s["table"][i, :-(-n // case["page"])].long()
            out[names] = _exact_bounds(_exact_sequence(s["k_pages"], s["table"][i], n, False), case["page"])
        return out
    new, cached = lengths
    page = case["page"]
    if case["op"] == "append":
        q, paged = [], case["bits"] == 16
        wide = s["table"].shape[1] * page
        out = {name: s[name + "_pages"].double() if paged else torch.zeros((case["batch"], case["kv_heads"], wide, case["dim"]), dtype=torch.float64, device="cuda")
               for name in ("k", "v")}
        out["bounds"] = s["bounds"].double()
        for i, (n, have) in enumerate(zip(new, cached)):
            first = 0 if s["cu"] is None else int(s["cu"][i])
            at = s["positions"][:, i] if s["cu"] is None else s["positions"][:, first:first + n]
            q.append(_exact_turn(_exact_rows(s, "q", i, n), s, at))
            rows = {"k": _exact_turn(_exact_rows(s, "k", i, n), s, at), "v": _exact_rows(s, "v", i, n).double()}
            place = torch.arange(have, have + n, device="cuda")
            for name, value in (("k", False), ("v", True)):
                held = rows[name] if paged else _exact_four_bits(rows[name])
                old = _exact_sequence(s[name + "_pages"], s["table"][i], have, value) if have else held[:0]
                if paged:
                    out[name][s["table"][i, place // page].long(), :, place % page] = held
                else:
                    out[name][i, :, :have + n] = torch.cat([old, held]).transpose(0, 1)
                if name == "k":
                    begin = have // page
                    names = s["table"][i, begin:-(-(have + n) // page)].long()
                    out["bounds"][names] = _exact_bounds(torch.cat([old, held])[begin * page:], page)
        out["q"] = torch.cat(q) if case["packed"] else torch.stack([x.transpose(0, 1) for x in q])
        out["lengths"] = s["lengths"] + torch.tensor(new, dtype=torch.int32, device="cuda")
        return out
    chosen, keys, out = [], [], []
    group, top, first, last = case["heads"] // case["kv_heads"], case["top"], case["first"], case["last"]
    for i, (n, have) in enumerate(zip(new, cached)):
        q = _exact_rows(s, "q", i, n).double()
        used = -(-have // page)
        names = s["table"][i, :used].long()
        bounds = s["bounds"][names].double()
        k, v = (_exact_pages(s[name][names], value) for name, value in (("k_pages", False), ("v_pages", True)))
        for j in range(n):
            seen = have - n + j + 1
            count = -(-seen // page)
            for head in range(case["kv_heads"]):
                x = q[j, head * group:(head + 1) * group]
                score = torch.stack([torch.maximum(y * bounds[:count, head, 0], y * bounds[:count, head, 1]).sum(-1) for y in x]).amax(0)
                kept = [e for e in range(count) if e < first or e >= count - last]
                free = [e for e in range(count) if first <= e < count - last]
                rest = min(len(free), top - len(kept)) if count > top else len(free)
                if rest < len(free):
                    best = torch.sort(score[free], descending=True, stable=True).indices[:rest].tolist()
                    free = sorted(free[e] for e in best)
                mine = sorted(kept + free)
                chosen.append(torch.nn.functional.pad(s["table"][i][torch.tensor(mine, device="cuda")], (0, top - len(mine)), value=-1))
                many = (len(mine) - 1) * page + (seen - 1) % page + 1
                keys.append(many)
                at = torch.tensor(mine, device="cuda")
                mk, mv = k[at, head].flatten(0, 1)[:many], v[at, head].flatten(0, 1)[:many]
                out.append(torch.softmax(x @ mk.T / math.sqrt(case["dim"]), dim=-1) @ mv)
    t = sum(new)
    out = torch.stack(out).view(t, case["heads"], case["dim"])
    if not case["packed"]:
        out = out.view(case["batch"], case["tokens"], case["heads"], case["dim"]).transpose(1, 2)
    return {"chosen": torch.stack(chosen).view(t, case["kv_heads"], top), "keys": torch.tensor(keys, dtype=torch.int32, device="cuda").view(t, case["kv_heads"]),
            "out": out}


# ---- what a pass cannot do without --------------------------------------------------------

def work(case):
    """Each input read and each output written once."""
    lengths = _lengths(case, 0)
    if case["op"] == "reserve":
        new, cached = lengths
        pages = sum(-(-(n + have) // case["page"]) - -(-have // case["page"]) for n, have in zip(new, cached))
        return {"bytes": 8 * pages + 12 * sum(new) + 16 * case["batch"] + 8, "flops": 0}
    d = case["dim"]
    if case["op"] == "rotary":
        tokens = case["tokens"] if case["packed"] else case["tokens"] * case["batch"]
        passes = 2 if case["grad"] else 1
        one = 4 if case["dtype"] == "fp32" else 2
        row = (case["heads"] + case["kv_heads"]) * d
        # (Each axis goes through its own positions of the tables, at most as many as there are tokens in a sequence.)
        places = max(lengths) if case["packed"] else case["tokens"]
        return {"bytes": passes * 2 * tokens * row * one + 4 * case["part"] * min(places, 4096) + 4 * case["axes"] * tokens,
                "flops": passes * 3 * tokens * (case["heads"] + case["kv_heads"]) * case["part"]}
    hk = case["kv_heads"]
    cell = hk * (2 * d if case["bits"] == 16 else d // 2 + d // 16)     # keys of a token in the pages
    edge = 4 * hk * d                                                     # bounds of a page
    if case["op"] == "bounds":
        pages = sum(-(-n // case["page"]) for n in lengths)
        return {"bytes": sum(lengths) * cell + pages * edge, "flops": 2 * sum(lengths) * hk * d}
    new, cached = lengths
    rows = sum(new) * case["heads"] * d * 2
    if case["op"] == "append":
        pages = sum(-(-(n + have) // case["page"]) - have // case["page"] for n, have in zip(new, cached))
        begun = sum(1 for have in cached if have % case["page"])
        nbytes = 2 * rows + sum(new) * (4 * hk * d + 2 * cell + 4 * case["axes"]) + 8 * case["batch"] + 4 * case["part"] * min(sum(new), 4096) + (pages + begun) * edge
        if case["bits"] == 4:
            places = case["batch"] * _wide(case) * case["page"]
            nbytes += sum(cached) * 2 * cell + places * 4 * hk * d
        return {"bytes": nbytes, "flops": 3 * sum(new) * (case["heads"] + hk) * case["part"] + 2 * sum(new) * hk * d}
    page, top = case["page"], case["top"]
    pages, keys, flops = 0, 0, 0
    for n, have in zip(new, cached):
        used = -(-have // page)
        pages += used
        keys += min(have, n * top * page)
        flops += n * case["heads"] * (4 * d * used + 4 * d * min(have, top * page))
    return {"bytes": 2 * rows + pages * edge + keys * 2 * cell + sum(new) * hk * 4 * (top + 1) + 4 * pages, "flops": flops}
