"""Test infrastructure: block tables out of a list of free pages, positions of several axes, bounds of pages, the pages that a
query selects and attention over them, on the CPU in float64 or whole numbers, written from their definitions."""

import math

import torch

from oracle import paged_oracle as po


def reserve(table, lengths, added, free, count, page, tokens):
    """(table, cu, positions, slots, granted, left) as lists, of lists and whole numbers."""
    table, width, left, short = [list(r) for r in table], len(table[0]), count, False
    cu, positions, slots, granted = [0], [], [], []
    for row, n, more in zip(table, lengths, added):
        n, more = min(max(n, 0), width * page), max(more, 0)
        held, wanted = -(-n // page), -(-(n + more) // page)
        short = short or wanted > width or wanted - held > left
        for e in range(held, min(wanted, width)):
            row[e] = -1
            if not short:
                left -= 1
                row[e] = free[left]
        places = list(range(n, n + more))
        cu.append(cu[-1] + more)
        positions += places
        slots += [-1 if short or row[p // page] < 0 else row[p // page] * page + p % page for p in places]
        granted.append(0 if short else more)
    positions, slots = positions[:tokens], slots[:tokens]
    return table, cu, positions + [-1] * (tokens - len(positions)), slots + [-1] * (tokens - len(slots)), granted, left


def append(contents, table, lengths, rows, granted):
    """New rows [n, Hk, D] of each sequence into bf16 `contents` [pages, Hk, page, D], in place, the first granted[b] of them; the new lengths."""
    pages, page, cap, after = contents.shape[0], contents.shape[2], table.shape[1] * contents.shape[2], []
    for b, (n, new, some) in enumerate(zip(lengths, rows, granted)):
        n = min(max(n, 0), cap)
        some = min(max(some, 0), len(new))
        for at, row in zip(range(n, min(n + some, cap)), new):
            if 0 <= table[b, at // page] < pages:
                contents[table[b, at // page], :, at % page] = row
        after.append(min(n + some, cap))
    return after


def release(table, lengths, kept, free, count, page):
    """(table, free, count) after it."""
    table, free, pool, width = [list(r) for r in table], list(free), len(free), len(table[0])
    for row, n, keep in zip(table, lengths, kept):
        n = min(max(n, 0), width * page)
        keep = min(max(keep, 0), n)
        for e in range(-(-keep // page), -(-n // page)):
            if 0 <= row[e] < pool:
                if count < pool:
                    free[count] = row[e]
                count += 1
            row[e] = -1
    return table, free, min(count, pool)


def axis_rows(cos, sin, positions, axes):
    """cos, sin [..., pairs] of positions [axes, ...], clamped to the tables."""
    at = positions.long().clamp(0, cos.shape[0] - 1)
    return (torch.stack([t[at[a], i] for i, a in enumerate(axes)], -1) for t in (cos, sin))


def bounds(k_pages, table, lengths, into, since=None):
    """`into` [pages, Hk, 2, D] with the pages that keys since[b] .. lengths[b] - 1 lie in, from all of their keys; bf16 keys as they
    are, 4 bits as bf16."""
    out, vals, page = into.clone(), po.values(k_pages, False).to(torch.bfloat16), k_pages.shape[2]
    for b, n in enumerate(lengths):
        n = min(max(n, 0), table.shape[1] * page)
        first = 0 if since is None else min(max(since[b], 0), n)
        for e in range(first // page, -(-n // page)) if first < n else ():
            name = int(table[b, e])
            if 0 <= name < k_pages.shape[0]:
                x = vals[name, :, :min(page, n - e * page)]
                bad = x.isnan().any(1)
                out[name, :, 0] = torch.where(bad, torch.nan, x.amin(1))
                out[name, :, 1] = torch.where(bad, torch.nan, x.amax(1))
    return out


def tokens(counts, lengths, cap):
    """(sequence, keys seen) of each token of sequences with `counts` query tokens."""
    out = []
    for b, (n, have) in enumerate(zip(counts, lengths)):
        have = min(max(have, 0), cap)
        out += [(b, max(0, have - n + i + 1)) for i in range(n)]
    return out


def select(q, bnds, table, owners, page, top, first, last):
    """chosen [T, Hk, top], keys [T, Hk] of queries [T, H, D]; owners: (sequence or -1, keys seen) of each."""
    t, h, d = q.shape
    pages, hk = bnds.shape[:2]
    chosen, keys = torch.full((t, hk, top), -1, dtype=torch.int32), torch.zeros((t, hk), dtype=torch.int32)
    q, bnds = q.double(), bnds.double()
    for i, (b, seen) in enumerate(owners):
        count = -(-seen // page)
        for head in range(hk):
            scores = []
            for e in range(count):
                name = int(table[b, e])
                if not 0 <= name < pages:
                    scores.append(0.0)
                    continue
                x, (lo, hi) = q[i, head * (h // hk):(head + 1) * (h // hk)], bnds[name, head]
                s = torch.maximum(x * lo, x * hi).sum(-1)
                scores.append(torch.where(s.isnan(), math.inf, s).max().item())
            kept = [e for e in range(count) if e < first or e >= count - last]
            rest = [e for e in range(count) if first <= e < count - last]
            if count > top:
                rest = sorted(sorted(rest, key=lambda e: (-scores[e], e))[:top - len(kept)])
            mine = sorted(kept + rest)
            chosen[i, head, :len(mine)] = torch.tensor([int(table[b, e]) for e in mine], dtype=torch.int32)
            if mine:
                keys[i, head] = (len(mine) - 1) * page + (seen - 1) % page + 1
    return chosen, keys


def attend(q, k_pages, v_pages, chosen, keys, scale):
    """Of queries [T, H, D] over tables of their own: (out, sum p (|v| + step |code - 8|), largest sum |q| |k| scale) as po.attend's."""
    t, h, d = q.shape
    group = h // chosen.shape[1]
    out, mag, size = torch.zeros((t, h, d), dtype=torch.float64), torch.zeros((t, h, d), dtype=torch.float64), torch.zeros((t, h), dtype=torch.float64)
    kv, vv, mid = po.values(k_pages, False), po.values(v_pages, True), po.about_middle(v_pages)
    cap = chosen.shape[2] * k_pages.shape[2]
    for i in range(t):
        for head in range(chosen.shape[1]):
            n = min(max(int(keys[i, head]), 0), cap)
            if n == 0:
                continue
            k, v = po.sequence(k_pages, chosen[i, head], n, False, kv)[head], po.sequence(v_pages, chosen[i, head], n, True, vv)[head]
            a = v.abs() + po.sequence(v_pages, chosen[i, head], n, True, mid)[head]
            for g in range(head * group, (head + 1) * group):
                x = q[i, g].double()
                p = torch.softmax(k @ x * scale, 0)
                out[i, g], mag[i, g] = p @ v, p @ a
                size[i, g] = (k.abs() @ x.abs()).max() * scale
    return out, mag, size
