"""Test infrastructure: rotary positions, a paged cache and attention over it in float64 on the CPU,
written from their definitions, and the layout of pages that hold 4 bits per value."""

import math

import torch


def table(positions, frequencies, scale=1.0):
    """float64 cos, sin [positions, pairs]."""
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * torch.tensor(frequencies, dtype=torch.float64)
    return scale * angle.cos(), scale * angle.sin()


def turn(x, cos, sin, interleaved, inverse=False):
    """x [..., D] float64, cos / sin [..., pairs]: the rotation, and what it could be off by in fp32 per
    2^-24 (the sum of its terms' magnitudes)."""
    x, cos, sin = x.double(), cos.double(), sin.double()
    if inverse:
        sin = -sin
    pairs = cos.shape[-1]
    y, size = x.clone(), x.abs().clone()
    for i in range(pairs):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        y[..., a] = x[..., a] * cos[..., i] - x[..., b] * sin[..., i]
        y[..., b] = x[..., b] * cos[..., i] + x[..., a] * sin[..., i]
        size[..., a] = (x[..., a] * cos[..., i]).abs() + (x[..., b] * sin[..., i]).abs()
        size[..., b] = (x[..., b] * cos[..., i]).abs() + (x[..., a] * sin[..., i]).abs()
    return y, size


def turn_fp32(x, cos, sin, interleaved):
    """The rotation in fp32 with every product and sum rounded, as the kernels define it; x's type."""
    pairs = cos.shape[-1]
    y, f = x.clone(), x.float()
    for i in range(pairs):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        c, s = cos[..., i], sin[..., i]
        y[..., a] = (f[..., a] * c - f[..., b] * s).to(x.dtype)
        y[..., b] = (f[..., b] * c + f[..., a] * s).to(x.dtype)
    return y


def nibble(dim, value, token, channel):
    """Which nibble of a block of 16 tokens holds the code of (token, channel)."""
    x, e = channel // 8, channel % 8
    if value:
        pair, g, groups = token // 2, x % 8, dim // 64
        place = g ^ (2 * (pair % 4)) if dim == 128 else g ^ (4 * (pair // 2 % 2))
        word = (pair * 8 + place) * 2 * groups + token % 2 * groups + x // 8
    else:
        word = token * (dim // 8) + x % 4 * (dim // 32) + x // 4
    return word * 8 + e // 2 + 4 * (e % 2)


_MAPS = {}


def places(dim, value):
    if (dim, value) not in _MAPS:
        _MAPS[dim, value] = torch.tensor([nibble(dim, value, t, c) for t in range(16) for c in range(dim)])
    return _MAPS[dim, value]


def quantise(x):
    """(codes, step, least) of bf16 values [..., D] by groups of 64, as the append defines them; a group
    with a NaN is NaN."""
    g = x.float().unflatten(-1, (-1, 64))
    least, most = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    step = ((most - least) * torch.tensor(1.0 / 15, dtype=torch.float32)).to(torch.bfloat16).float()
    code = torch.where(step > 0, torch.round((g - least) / step), torch.zeros_like(g)).nan_to_num(0.0).clamp(0, 15)
    return code.flatten(-2), step.squeeze(-1), least.squeeze(-1)


def worth(code, step, least):
    """fp32 values of codes [..., D]."""
    return (least.unsqueeze(-1) + step.unsqueeze(-1) * code.unflatten(-1, (-1, 64))).flatten(-2)


def pack(x, value):
    """bf16 [pages, Hk, page, D] as uint8 pages of 4 bits."""
    n, hk, page, d = x.shape
    code, step, least = quantise(x)
    flat = torch.zeros((n, hk, page // 16, 16 * d), dtype=torch.uint8)
    flat[..., places(d, value)] = code.reshape(n, hk, page // 16, 16 * d).to(torch.uint8)
    codes = flat[..., 0::2] | flat[..., 1::2] << 4
    words = torch.stack([step, least], -1).to(torch.bfloat16).view(torch.uint8).reshape(n, hk, page // 16, d)
    return torch.cat([codes, words], -1).reshape(n, hk, page, d // 2 + d // 16)


def unpack(pages, value):
    """(codes, step, least) of uint8 pages."""
    n, hk, page, wide = pages.shape
    d = wide // 9 * 16
    blocks = pages.reshape(n, hk, page // 16, 16 * wide)
    codes, words = blocks[..., :8 * d], blocks[..., 8 * d:].contiguous()
    flat = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    code = flat[..., places(d, value)].reshape(n, hk, page, d).float()
    pair = words.view(torch.bfloat16).reshape(n, hk, page, d // 64, 2).float()
    return code, pair[..., 0], pair[..., 1]


def values(pages, value):
    """fp32 [pages, Hk, page, D] that pages of either kind stand for."""
    return worth(*unpack(pages, value)) if pages.dtype == torch.uint8 else pages.float()


def about_middle(pages):
    """What pages of 4 bits hold beside the middle of their range: step * |code - 8|; 0 for bf16."""
    if pages.dtype != torch.uint8:
        return torch.zeros_like(pages, dtype=torch.float32)
    code, step, _ = unpack(pages, True)
    return worth(code - 8, step, torch.zeros_like(step)).abs()


def sequence(pages, row, count, value, vals=None):
    """float64 [Hk, count, D]; zeros where there is no page."""
    page = pages.shape[2]
    vals = (values(pages, value) if vals is None else vals).double()
    got = torch.zeros((pages.shape[1], count, vals.shape[-1]), dtype=torch.float64)
    for j in range(count):
        p = int(row[j // page])
        if 0 <= p < pages.shape[0]:
            got[:, j] = vals[p, :, j % page]
    return got


def attend(q, k_pages, v_pages, table_rows, lengths, causal, scale, counts=None):
    """q: list of [H, n, D] float64 per sequence. Returns lists (out, sum p (|v| + step |code - 8|), largest
    sum |q| |k| scale per row) per sequence."""
    outs, mags, sizes = [], [], []
    cap = table_rows.shape[1] * k_pages.shape[2]
    for b, x in enumerate(q):
        h, n, d = x.shape
        length = min(max(int(lengths[b]), 0), cap)
        k, v = sequence(k_pages, table_rows[b], length, False), sequence(v_pages, table_rows[b], length, True)
        a = v.abs() + sequence(v_pages, table_rows[b], length, True, about_middle(v_pages))
        group = h // k.shape[0]
        o, m, z = torch.zeros_like(x), torch.zeros_like(x), torch.zeros((h, n), dtype=torch.float64)
        for i in range(n):
            last = min(length, length - n + i + 1) if causal else length
            if last <= 0:
                continue
            for head in range(h):
                kk, vv, aa = k[head // group][:last], v[head // group][:last], a[head // group][:last]
                logits = kk @ x[head, i] * scale
                p = torch.softmax(logits, 0)
                o[head, i], m[head, i] = p @ vv, p @ aa
                z[head, i] = (kk.abs() @ x[head, i].abs()).max() * abs(scale)
        outs.append(o)
        mags.append(m)
        sizes.append(z)
    return outs, mags, sizes


def turns_within(frequency, original):
    return original * frequency / (2 * math.pi)
