"""The work that the operators around a paged cache of keys and values are timed on: rotary
positions, the append to the cache, reading it back, and attention over it.

A case is a dict of plain values; `op` says which operator it goes through:

    "table"    rotary_table: cosines and sines of every position, scaled for long contexts or not
    "rotary"   rotary of queries and keys, alone or with its gradients
    "append"   paged_append: rotation of queries and keys, new rows into the pages
    "read"     paged_read: the pages as dense keys and values
    "attend"   sdpa_paged: attention over the pages, of single tokens, a few, or chunks of prompts

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


def _table(positions, dim, scaling, factor=1.0, original=0, base=10000.0):
    return {"op": "table", "positions": positions, "dim": dim, "scaling": scaling, "factor": factor, "original": original, "base": base}


def _rotary(batch, heads, kv_heads, tokens, dim, part, interleaved, grad, packed=False, dtype="bf16"):
    """`tokens` of each sequence, or of the packed batch; `part`: the columns that turn."""
    return {"op": "rotary", "batch": batch, "heads": heads, "kv_heads": kv_heads, "tokens": tokens, "dim": dim, "part": part,
            "interleaved": interleaved, "grad": grad, "packed": packed, "dtype": dtype}


def _append(bits, batch, heads, kv_heads, tokens, keys, dim, part, interleaved, page, packed=False):
    """`tokens` new ones of each sequence (packed: at most) behind up to `keys` cached ones."""
    return {"op": "append", "bits": bits, "batch": batch, "heads": heads, "kv_heads": kv_heads, "tokens": tokens, "keys": keys,
            "dim": dim, "part": part, "interleaved": interleaved, "page": page, "packed": packed}


def _read(bits, batch, kv_heads, keys, dim, page):
    return {"op": "read", "bits": bits, "batch": batch, "kv_heads": kv_heads, "keys": keys, "dim": dim, "page": page}


def _attend(bits, batch, heads, kv_heads, tokens, keys, dim, page, packed=False):
    """`tokens` queries of each sequence (packed: at most) over up to `keys` keys, these queries' own among them."""
    return {"op": "attend", "bits": bits, "batch": batch, "heads": heads, "kv_heads": kv_heads, "tokens": tokens, "keys": keys,
            "dim": dim, "page": page, "packed": packed}


def _draw_table(rng):
    scaling = rng.choice(["none", "linear", "base", "parts"])
    return _table(_spread(rng, 1024, 131072), 2 * rng.randint(16, 64), scaling, factor=round(rng.uniform(2, 32), 2), original=_spread(rng, 1024, 8192),
                  base=rng.choice([10000.0, 500000.0, 1000000.0]))


def _draw_rotary(rng):
    h, hk = rng.choice(GROUPED + PLAIN)
    d = rng.choice([64, 80, 96, 128])
    part = rng.choice([d, d, d // 2, 2 * rng.randint(4, d // 2)])
    tokens = _spread(rng, 1, 65536)
    batch = _spread(rng, 1, max(1, min(64, 65536 // tokens)))
    packed = rng.random() < 0.4
    return _rotary(batch, h, hk, tokens, d, part, rng.random() < 0.4, rng.random() < 0.5, packed, rng.choice(["bf16", "bf16", "fp16", "fp32"]))


def _draw_append(rng):
    h, hk = rng.choice(GROUPED + PLAIN)
    d = rng.choice([64, 128])
    packed = rng.random() < 0.6
    tokens = _spread(rng, 8, 2048) if packed else rng.choice([1, 1, 1, _spread(rng, 2, 256)])
    keys = _spread(rng, 64, 4096)
    batch = _spread(rng, 1, max(1, min(64, 8192 // tokens, 131072 // (tokens + keys))))
    return _append(rng.choice([16, 4]), batch, h, hk, tokens, keys, d, rng.choice([d, d, d // 2]), rng.random() < 0.3, rng.choice([16, 32, 64]), packed)


def _draw_read(rng):
    _, hk = rng.choice(GROUPED + PLAIN)
    keys = _spread(rng, 64, 16384)
    return _read(rng.choice([16, 4]), _spread(rng, 1, max(1, min(64, 65536 // keys))), hk, keys, rng.choice([64, 128]), rng.choice([16, 32, 64]))


def _draw_attend(rng):
    h, hk = rng.choice(GROUPED + PLAIN)
    tokens = rng.choice([1, 1, 1, rng.randint(2, 8), _spread(rng, 16, 1024)])
    keys = max(_spread(rng, 128, 16384), 2 * tokens)
    batch = _spread(rng, 1, max(1, min(64, 2097152 // (keys * hk), 1 << 23, (1 << 27) // (tokens * keys * h) if tokens > 8 else 64)))
    return _attend(rng.choice([16, 4]), batch, h, hk, tokens, keys, rng.choice([64, 128]), rng.choice([16, 32, 64, 128]), tokens > 8 and rng.random() < 0.5)


FAMILIES = [
    # Loading a model: its rotary tables, of a short context and of one stretched eight times by parts.
    ([dict(_table(4096, 64, "none"), name="table"),
      dict(_table(131072, 128, "parts", factor=8.0, original=16384, base=1000000.0), name="table stretched")], _draw_table),
    # A short prompt of an odd length before its attention; and a training step on packed sequences, half of
    # each head turning in pairs of neighbours: the largest pass.
    ([dict(_rotary(1, 14, 2, 77, 64, 64, False, False), name="rotary short"),
      dict(_rotary(16, 16, 16, 65536, 128, 64, True, True, packed=True), name="rotary train")], _draw_rotary),
    # The neighbours of a token of a full server batch; and prompts of many lengths whose cache is kept in 4
    # bits, some of them behind a prefix that is cached already, with the check that a server makes of it: the
    # cache read back.
    ([dict(_append(16, 64, 16, 2, 1, 1024, 128, 128, False, 16), name="append token"),
      dict(_append(4, 8, 32, 8, 2048, 2048, 128, 128, False, 16, packed=True), name="append prompts")], _draw_append),
    # A cached prefix handed to a program that wants plain tensors.
    ([dict(_read(4, 4, 8, 8192, 128, 16), name="read")], _draw_read),
    # Generating text: one sequence, one new token, a short cache in bf16 (the least there is) and a long one in
    # 4 bits; a full server batch over both; and prompts read in chunks behind what is cached.
    ([dict(_attend(16, 1, 14, 2, 1, 1024, 64, 16), name="attend one"),
      dict(_attend(4, 1, 32, 8, 1, 32768, 128, 64), name="attend one long, 4 bits"),
      dict(_attend(16, 64, 16, 2, 1, 4096, 128, 16), name="attend batch"),
      dict(_attend(4, 64, 16, 2, 1, 16384, 128, 16), name="attend batch, 4 bits"),
      dict(_attend(4, 4, 16, 4, 512, 8192, 128, 32, packed=True), name="attend chunks, 4 bits")], _draw_attend),
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
    family = rng.choice([_draw_table, _draw_rotary, _draw_rotary, _draw_append, _draw_append, _draw_read, _draw_attend, _draw_attend, _draw_attend])
    while True:
        case = family(rng)
        if _cost(case) <= _most():
            return case


# ---- the pages --------------------------------------------------------------------------

@functools.lru_cache(None)
def _places(dim, value):
    """[16, D]: which nibble of a block holds the code of (token, channel). Eight channels share a word of 32
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


def _dense(pages, table, value):
    """fp32 [B, Hk, rows, D] of the pages that a table names (those that it names none for: page 0)."""
    got = pages[table.clamp(min=0).long()].transpose(1, 2)
    got = _values(*_parts_of(got, value)) if pages.dtype == torch.uint8 else got.float()
    return got.flatten(2, 3)


# ---- inputs -----------------------------------------------------------------------------

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _lengths(case, seed):
    """What the sequences of a case have: ("table": none) the tokens of each (packed rotary), or the new tokens
    of each and the keys that are cached (append: before them; read, attend: in all), uniform over the range."""
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
    if case["op"] == "read":
        return cached
    new = [case["tokens"]] * b
    if case["packed"]:   # each sequence with an opposite, so that all seeds have as many tokens
        low, high = max(1, case["tokens"] // 4), case["tokens"]
        new = of(low, high, b // 2)
        new += [low + high - n for n in new] + [(low + high) // 2] * (b % 2)
    if case["op"] == "append":
        cached = [0 if i % 2 and case["packed"] else x for i, x in enumerate(cached)]
    else:
        cached = [max(x, y) for x, y in zip(cached, new)]
    return new, cached


def _normal(g, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _tables(positions, part, base=10000.0):
    """The plan that a program keeps: fp32 cosines and sines."""
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * base ** (-torch.arange(0, part, 2, device="cuda", dtype=torch.float64) / part)
    return angle.cos().float(), angle.sin().float()


def _cumulative(lengths):
    return torch.tensor([0] + lengths).cumsum(0).to(device="cuda", dtype=torch.int32)


def _wide(case):
    """Pages that a sequence may have."""
    return -(-(case["keys"] + (case["tokens"] if case["op"] == "append" else 0)) // case["page"])


def _cache(g, case, rows):
    """A pool of pages filled with rows of the distribution of keys and values, and a table that names pages in
    no order for the `rows` of each sequence, and none behind them."""
    b, hk, d, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    used, wide = [-(-n // page) for n in rows], _wide(case)
    count = b * wide
    names = torch.randperm(count, generator=g, device="cuda").to(torch.int32)
    table = torch.full((b, wide), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = names[at:at + n]
        at += n

    def pages(value):
        if case["bits"] == 16:
            return _normal(g, count, hk, page, d)
        return torch.cat([_pack(_normal(g, min(2048, count - i), hk, page, d), value) for i in range(0, count, 2048)])

    return pages(False), pages(True), table


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "table":
        # The seed decides the base, by a little: another one is another table.
        state["base"] = case["base"] * (1 + 1e-3 * (seed % 997))
        return state
    lengths, d = _lengths(case, seed), case["dim"]
    if case["op"] == "rotary":
        n, dtype = case["tokens"], DTYPES[case["dtype"]]
        if case["packed"]:
            state["positions"] = torch.cat([torch.arange(x) for x in lengths]).to(device="cuda", dtype=torch.int32)
            shapes = [(n, case["heads"], d), (n, case["kv_heads"], d)]
        else:
            state["positions"] = None
            shapes = [(case["batch"], case["heads"], n, d), (case["batch"], case["kv_heads"], n, d)]
        state["cos"], state["sin"] = _tables(n if lengths is None else max(lengths), case["part"])
        state["q"], state["k"] = (_normal(g, *s, dtype=dtype).requires_grad_(case["grad"]) for s in shapes)
        if case["grad"]:
            state["dq"], state["dk"] = (_normal(g, *s, dtype=dtype) for s in shapes)
        return state
    if case["op"] == "read":
        state["k_pages"], state["v_pages"], state["table"] = _cache(g, case, lengths)
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        return state
    new, cached = lengths
    append = case["op"] == "append"
    state["k_pages"], state["v_pages"], state["table"] = _cache(g, case, [x + y for x, y in zip(new, cached)] if append else cached)
    state["lengths"] = torch.tensor(cached, dtype=torch.int32, device="cuda")
    state["cu"], state["max_q"] = (_cumulative(new), max(new)) if case["packed"] else (None, None)
    n, h, hk, b = sum(new), case["heads"], case["kv_heads"], case["batch"]
    state["q"] = _normal(g, n, h, d) if case["packed"] else _normal(g, b, h, case["tokens"], d)
    if append:
        shape = (n, hk, d) if case["packed"] else (b, hk, case["tokens"], d)
        state["k"], state["v"] = _normal(g, *shape), _normal(g, *shape)
        state["cos"], state["sin"] = _tables(state["table"].shape[1] * case["page"], case["part"])
        state["next"] = torch.empty_like(state["lengths"])
    return state


# ---- one pass ---------------------------------------------------------------------------

def _plain_table(case, base):
    r, factor = case["dim"], case["factor"]
    if case["scaling"] == "base":
        base = base * factor ** (r / (r - 2))
    f = base ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
    scale = 1.0
    if case["scaling"] == "linear":
        f = f / factor
    elif case["scaling"] == "parts":
        keep = ((case["original"] * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = (1 - keep) * f / factor + keep * f
        scale = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(case["positions"], device="cuda", dtype=torch.float64)[:, None] * f
    return {"cos": (angle.cos() * scale).float(), "sin": (angle.sin() * scale).float()}


def _turn(x, cos, sin, interleaved):
    """fp32 rotation of the first columns of x [..., D] by cos, sin [..., R / 2]; rounded to x's type."""
    r = 2 * cos.shape[-1]
    head, rest = x[..., :r].float(), x[..., r:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else head.chunk(2, dim=-1)
    y1, y2 = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([y1, y2], dim=-1).flatten(-2) if interleaved else torch.cat([y1, y2], dim=-1)
    return torch.cat([y.to(x.dtype), rest], dim=-1)


def _plain_rotary(s):
    case, cos, sin = s["case"], s["cos"], s["sin"]
    if case["packed"]:
        at = s["positions"].long()
        cos, sin = cos[at][:, None], sin[at][:, None]
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


def _plain_append(s):
    case, page, d = s["case"], s["case"]["page"], s["case"]["dim"]
    if case["packed"]:
        seq, place = _rows_of(s, s["q"].shape[0])
        at = s["lengths"].long()[seq] + place
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
        k_rows, v_rows = _turn(s["k"], cos, sin, case["interleaved"]), s["v"]
        added = s["cu"][1:] - s["cu"][:-1]
    else:
        b, n = case["batch"], case["tokens"]
        at = s["lengths"].long()[:, None] + torch.arange(n, device="cuda")
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
        k_rows, v_rows = (x.transpose(1, 2).flatten(0, 1) for x in (_turn(s["k"], cos, sin, case["interleaved"]), s["v"]))
        seq, at = torch.arange(b, device="cuda").repeat_interleave(n), at.flatten()
        added = n
    q = _turn(s["q"], cos, sin, case["interleaved"])
    to, row = s["table"][seq, at // page].long(), at % page
    s["next"].copy_(s["lengths"] + added)
    out = {"q": q, "lengths": s["next"]}
    for name, rows, value in (("k", k_rows, False), ("v", v_rows, True)):
        pages = s[name + "_pages"]
        if case["bits"] == 16:
            pages[to, :, row] = rows
            out[name] = pages
            continue
        code, step, least = _parts_of(pages, value)
        new = _quantise(rows.float())
        for have, want in zip((code, step, least), new):
            have[to, :, row] = want
        wide = s["table"].shape[1] * page
        there = (torch.arange(wide, device="cuda") < s["next"][:, None])[:, None, :, None]
        got = _values(code, step, least)[s["table"].clamp(min=0).long()].transpose(1, 2).flatten(2, 3)
        out[name] = torch.where(there, got, torch.zeros_like(got)).to(torch.bfloat16)
    return out


def _plain_read(s):
    k, v = _dense(s["k_pages"], s["table"], False), _dense(s["v_pages"], s["table"], True)
    there = (torch.arange(k.shape[2], device="cuda") < s["lengths"][:, None])[:, None, :, None]
    return {"k": torch.where(there, k, torch.zeros_like(k)).to(torch.bfloat16), "v": torch.where(there, v, torch.zeros_like(v)).to(torch.bfloat16)}


def _plain_attend(s):
    case, d = s["case"], s["case"]["dim"]
    k, v = _dense(s["k_pages"], s["table"], False), _dense(s["v_pages"], s["table"], True)
    q = s["q"].float()
    if case["packed"]:   # padded to the longest
        seq, place = _rows_of(s, q.shape[0])
        added = s["cu"][1:] - s["cu"][:-1]
        rows = torch.zeros((case["batch"], case["tokens"], case["heads"], d), device="cuda")
        rows[seq, place] = q
        q = rows.transpose(1, 2)
    else:
        added = case["tokens"]
    b, h, n, _ = q.shape
    hk, keys = k.shape[1], k.shape[2]
    logits = (q.reshape(b, hk, h // hk * n, d) @ k.transpose(-1, -2)).reshape(b, hk, h // hk, n, keys) / math.sqrt(d)
    last = (s["lengths"] - added)[:, None] + torch.arange(n, device="cuda")     # the last key that a row sees
    seen = (torch.arange(keys, device="cuda") <= last[..., None])[:, None, None]
    logits = torch.where(seen, logits, torch.full_like(logits, -math.inf))
    most = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(most == -math.inf, torch.zeros_like(most), most))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    out = (p.reshape(b, hk, h // hk * n, keys) @ v).reshape(b, h, n, d)
    if case["packed"]:
        out = out.transpose(1, 2)[seq, place]
    return out.to(torch.bfloat16)


def run(s):
    case = s["case"]
    if not own:
        if case["op"] == "table":
            return _plain_table(case, s["base"])
        with torch.no_grad():
            return {"rotary": _plain_rotary, "append": _plain_append, "read": _plain_read, "attend": _plain_attend}[case["op"]](s)
    ktt = _ktt()
    if case["op"] == "table":
        scaling = None if case["scaling"] == "none" else case["scaling"]
        cos, sin = ktt.rotary_table(case["positions"], case["dim"], base=s["base"], scaling=scaling, factor=case["factor"], original=case["original"],
                                    device="cuda")
        return {"cos": cos, "sin": sin}
    if case["op"] == "rotary":
        q, k = ktt.rotary(s["q"], s["k"], s["cos"], s["sin"], positions=s["positions"], interleaved=case["interleaved"])
        if not case["grad"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if case["op"] == "append":
        q = ktt.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], cos=s["cos"], sin=s["sin"], q=s["q"],
                             interleaved=case["interleaved"], cu_seq=s["cu"], lengths_out=s["next"])
        if case["bits"] == 16:
            return {"q": q, "lengths": s["next"], "k": s["k_pages"], "v": s["v_pages"]}
        k, v = ktt.paged_read(s["k_pages"], s["v_pages"], s["table"], s["next"])
        return {"q": q, "lengths": s["next"], "k": k, "v": v}
    if case["op"] == "read":
        k, v = ktt.paged_read(s["k_pages"], s["v_pages"], s["table"], s["lengths"])
        return {"k": k, "v": v}
    return ktt.sdpa_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], is_causal=True, cu_seq_q=s["cu"], max_q=s["max_q"])


# ---- the definition in 64 bits ----------------------------------------------------------

def _exact_turn(x, cos, sin, interleaved):
    """x [n, H, D] turned by cos, sin [n, R / 2], as complex numbers; nothing rounded."""
    x, r = x.double(), 2 * cos.shape[-1]
    turn = torch.complex(cos.double(), sin.double())[:, None]
    y = x.clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(x[..., first], x[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rows(s, name, i, n):
    """Row-major [n, heads, D] of sequence i."""
    if s["cu"] is None:
        return s[name][i].transpose(0, 1)
    at = int(s["cu"][i])
    return s[name][at:at + n]


def _exact_sequence(pages, table, n, value):
    """The first n rows of a sequence, [n, Hk, D] in 64 bits, from its pages."""
    page = pages.shape[2]
    got = pages[table[:-(-n // page)].long()]
    if pages.dtype == torch.uint8:
        code, step, least = (x.double() for x in _parts_of(got, value))
        got = least.repeat_interleave(64, -1) + step.repeat_interleave(64, -1) * code
    return got.double().transpose(1, 2).flatten(0, 1)[:n]


def _exact_four_bits(x):
    """What a row [n, Hk, D] of bf16 values is worth once it is held in 4 bits."""
    x = x.to(torch.bfloat16).double().unflatten(-1, (-1, 64))
    least, most = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step = ((most - least) / 15).to(torch.bfloat16).double()
    return (least + step * torch.round((x - least) / step.clamp(min=1e-300)).clamp(0, 15)).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "table":
        r, factor, base = case["dim"], case["factor"], s["base"]
        pos, out = torch.arange(case["positions"], dtype=torch.float64, device="cuda"), []
        for i in range(r // 2):
            f, scale = math.exp(-2 * i / r * math.log(base)), 1.0
            if case["scaling"] == "base":
                f = math.exp(-2 * i / r * (math.log(base) + r / (r - 2) * math.log(factor)))
            elif case["scaling"] == "linear":
                f /= factor
            elif case["scaling"] == "parts":
                turns = case["original"] * f / (2 * math.pi)
                keep = min(1.0, max(0.0, (turns - 1) / 31))
                f, scale = f * (keep + (1 - keep) / factor), 1 + math.log(factor) / 10
            out.append(torch.polar(torch.full_like(pos, scale), pos * f))
        out = torch.stack(out, dim=-1)
        return {"cos": out.real.contiguous(), "sin": out.imag.contiguous()}
    if case["op"] == "rotary":
        n = case["tokens"]
        at = s["positions"].long() if case["packed"] else torch.arange(n, device="cuda")
        cos, sin = s["cos"][at], s["sin"][at]
        out = {}
        for name in ("q", "k", "dq", "dk") if case["grad"] else ("q", "k"):
            x, turn = s[name].detach(), -sin if name[0] == "d" else sin
            if case["packed"]:
                out[name] = _exact_turn(x, cos, turn, case["interleaved"])
            else:
                out[name] = torch.stack([_exact_turn(y.transpose(0, 1), cos, turn, case["interleaved"]).transpose(0, 1) for y in x])
        return out
    if case["op"] == "read":
        out = {}
        for name, value in (("k", False), ("v", True)):
            pages = s[name + "_pages"]
            out[name] = torch.zeros((case["batch"], case["kv_heads"], s["table"].shape[1] * case["page"], case["dim"]), dtype=torch.float64, device="cuda")
            for i, n in enumerate(s["lengths"].tolist()):
                out[name][i, :, :n] = _exact_sequence(pages, s["table"][i], n, value).transpose(0, 1)
        return out
    new, cached = _lengths(case, seed)
    if case["op"] == "append":
        q, page = [], case["page"]
        paged = case["bits"] == 16
        wide = s["table"].shape[1] * page
        out = {name: s[name + "_pages"].double() if paged else torch.zeros((case["batch"], case["kv_heads"], wide, case["dim"]), dtype=torch.float64, device="cuda")
               for name in ("k", "v")}
        for i, (n, have) in enumerate(zip(new, cached)):
            at = torch.arange(have, have + n, device="cuda")
            cos, sin = s["cos"][at], s["sin"][at]
            q.append(_exact_turn(_exact_rows(s, "q", i, n), cos, sin, case["interleaved"]))
            rows = {"k": _exact_turn(_exact_rows(s, "k", i, n), cos, sin, case["interleaved"]), "v": _exact_rows(s, "v", i, n).double()}
            for name, value in (("k", False), ("v", True)):
                if paged:
                    out[name][s["table"][i, at // page].long(), :, at % page] = rows[name]
                else:
                    if have:
                        out[name][i, :, :have] = _exact_sequence(s[name + "_pages"], s["table"][i], have, value).transpose(0, 1)
                    out[name][i, :, have:have + n] = _exact_four_bits(rows[name]).transpose(0, 1)
        out["q"] = torch.cat(q) if case["packed"] else torch.stack([x.transpose(0, 1) for x in q])
        out["lengths"] = s["lengths"] + torch.tensor(new, dtype=torch.int32, device="cuda")
        return out
    out = []
    for i, (n, have) in enumerate(zip(new, cached)):
        k, v = (_exact_sequence(s[name], s["table"][i], have, value).transpose(0, 1) for name, value in (("k_pages", False), ("v_pages", True)))
        q = _exact_rows(s, "q", i, n).double().transpose(0, 1)
        group = case["heads"] // case["kv_heads"]
        seen = torch.ones((n, have), dtype=torch.bool, device="cuda").tril(have - n)
        got = []
        for head in range(case["heads"]):
            logits = (q[head] @ k[head // group].T / math.sqrt(case["dim"])).masked_fill(~seen, -math.inf)
            got.append(torch.softmax(logits, dim=-1) @ v[head // group])
        out.append(torch.stack(got, dim=1))
    return torch.cat(out) if case["packed"] else torch.stack([x.transpose(0, 1) for x in out])


# ---- what a pass cannot do without --------------------------------------------------------

def work(case):
    """Each input read and each output written once."""
    if case["op"] == "table":
        n = case["positions"] * case["dim"] // 2
        return {"bytes": 8 * n, "flops": 3 * n}
    lengths, d = _lengths(case, 0), case["dim"]
    if case["op"] == "rotary":
        tokens = case["tokens"] if case["packed"] else case["tokens"] * case["batch"]
        passes = 2 if case["grad"] else 1
        one = 4 if case["dtype"] == "fp32" else 2
        row = (case["heads"] + case["kv_heads"]) * d
        places = max(lengths) if case["packed"] else case["tokens"]
        return {"bytes": passes * 2 * tokens * row * one + 4 * case["part"] * places + (4 * tokens if case["packed"] else 0),
                "flops": passes * 3 * tokens * (case["heads"] + case["kv_heads"]) * case["part"]}
    hk = case["kv_heads"]
    cell = 2 * hk * (2 * d if case["bits"] == 16 else d // 2 + d // 16)     # keys and values of a token in the pages
    if case["op"] == "read":
        places = case["batch"] * _wide(case) * case["page"]
        return {"bytes": sum(lengths) * cell + places * 4 * hk * d, "flops": sum(lengths) * 2 * hk * d}
    new, cached = lengths
    rows = sum(new) * case["heads"] * d * 2
    if case["op"] == "append":
        nbytes = 2 * rows + sum(new) * (4 * hk * d + cell) + 8 * case["batch"] + 4 * case["part"] * len({x for n, have in zip(new, cached) for x in range(have, have + n)})
        if case["bits"] == 4:
            places = case["batch"] * _wide(case) * case["page"]
            nbytes += sum(cached) * cell + places * 4 * hk * d
        return {"bytes": nbytes, "flops": 3 * sum(new) * (case["heads"] + hk) * case["part"]}
    pairs = sum(n * have - n * (n - 1) // 2 for n, have in zip(new, cached))
    return {"bytes": 2 * rows + sum(cached) * cell + 4 * case["batch"], "flops": 4 * d * case["heads"] * pairs}
