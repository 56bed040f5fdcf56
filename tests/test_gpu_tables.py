"""Block tables on the device: pages out of a list of free ones, slots and positions, and pages given back."""

import random

import pytest
import torch

import kohaku_tt_b200 as ktt
from kohaku_tt_b200 import _lib
from oracle import serving_oracle as so

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    """Through the C++ edge, and through Python's."""
    if request.param == "python":
        monkeypatch.setattr(_lib, "_NATIVE", False)


def _i32(x, cuda):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


def _state(rng, batch, width, page, lengths, spare):
    """A table whose rows have pages for their lengths, and the list of the others."""
    held = [-(-n // page) for n in lengths]
    pool = sum(held) + spare
    names = list(range(pool))
    rng.shuffle(names)
    table = [[-1] * width for _ in range(batch)]
    for row, n in zip(table, held):
        for e in range(n):
            row[e] = names.pop()
    return table, names + [-7] * sum(held), len(names)


def _reserve(cuda, table, lengths, added, free, count, page, tokens):
    td, fd = _i32(table, cuda), _i32(free, cuda)
    left, n = torch.full((1,), -9, dtype=torch.int32, device=cuda), _i32([count], cuda)
    cu, positions, slots, granted = ktt.paged_reserve(td, _i32(lengths, cuda), _i32(added, cuda), fd, n, page, tokens, left)
    assert fd.tolist() == free and n.item() == count and slots.dtype == torch.int64 and positions.dtype == cu.dtype == granted.dtype == torch.int32
    return td.tolist(), cu.tolist(), positions.tolist(), slots.tolist(), granted.tolist(), left.item()


CASES = [  # batch, width, page, longest cached, most added, spare pages, rows more than there are
    (1, 1, 16, 0, 1, 1, 0), (1, 4, 16, 16, 1, 3, 0), (3, 8, 16, 40, 0, 5, 4), (5, 40, 32, 300, 70, 60, 1), (64, 20, 16, 250, 1, 40, 0), (64, 300, 16, 600, 900, 4000, 0),
    (257, 6, 48, 100, 60, 400, 3), (1000, 5, 16, 40, 30, 1500, 0), (4096, 2, 16, 16, 3, 4096, 0), (7, 9, 256, 2000, 256, 9, 0),
]


@pytest.mark.parametrize("batch,width,page,keys,added,spare,more", CASES)
def test_reserve(cuda, path, batch, width, page, keys, added, spare, more):
    for seed, room in ((0, spare), (1, spare // 3), (2, 0)):      # enough pages, too few for some, none
        rng = random.Random(seed * 100 + batch)
        lengths = [rng.randint(0, min(keys, width * page)) for _ in range(batch)]
        new = [rng.choice([0, rng.randint(0, added)]) for _ in range(batch)]
        table, free, count = _state(rng, batch, width, page, lengths, room)
        tokens = sum(new) + more
        want = so.reserve(table, lengths, new, free, count, page, tokens)
        assert _reserve(cuda, table, lengths, new, free, count, page, tokens) == tuple(want)


def test_reserve_at_the_edges(cuda, path):
    """Past a row of the table, lengths and counts out of range, fewer rows than there are, no rows at all."""
    table, free = [[3, -1], [-1, -1], [-1, -1]], [9, 8, 7, 6, 5]
    for lengths, new, count, tokens in (([16, 0, 0], [17, 1, 1], 5, 19), ([16, 0, 0], [16, 32, 1], 5, 49), ([16, 0, 0], [16, 33, 1], 5, 50), ([16, 0, 0], [1, 1, 1], 5, 2),
                                        ([16, 0, 0], [1, 1, 1], 5, 0), ([-4, -1, 0], [2, 3, 4], 5, 9), ([99, 0, 0], [1, 1, 0], 5, 2), ([99, 0, 0], [0, 20, 0], 5, 20),
                                        ([16, 0, 0], [-3, 5, -1], 5, 6)):
        want = so.reserve(table, lengths, new, free, count, 16, tokens)
        assert _reserve(cuda, table, lengths, new, free, count, 16, tokens) == tuple(want)
    for count in (-3, 0, 5, 77):      # (taken as 0 to the list's length)
        want = so.reserve(table, [16, 0, 0], [1, 40, 2], free, min(max(count, 0), 5), 16, 43)
        assert _reserve(cuda, table, [16, 0, 0], [1, 40, 2], free, count, 16, 43) == tuple(want)
    # A place whose page is missing has no slot.
    assert _reserve(cuda, [[-1, -1]], [5], [3], [9], 1, 16, 3)[3] == [-1, -1, -1]


@pytest.mark.parametrize("batch,width,page,keys", [(1, 1, 16, 16), (3, 8, 16, 128), (64, 40, 16, 640), (64, 700, 16, 11000), (4096, 2, 16, 32), (300, 11, 64, 700)])
def test_release(cuda, path, batch, width, page, keys):
    for seed in range(3):
        rng = random.Random(seed * 100 + batch)
        lengths = [rng.randint(0, keys) for _ in range(batch)]
        table, free, count = _state(rng, batch, width, page, lengths, 5)
        kept = [rng.choice([0, n, rng.randint(0, n), n + 3, -1]) for n in lengths]
        if seed == 1:      # entries that name no page, and a list that is too short
            for row in table:
                row[rng.randrange(width)] = rng.choice([-1, len(free), 1 << 30])
            free = free[:max(count, len(free) - 4)]
        want = so.release(table, lengths, kept, free, count, page)
        td, fd, left = _i32(table, cuda), _i32(free, cuda), torch.full((1,), -9, dtype=torch.int32, device=cuda)
        ktt.paged_release(td, _i32(lengths, cuda), _i32(kept, cuda), fd, _i32([count], cuda), page, left)
        assert (td.tolist(), fd.tolist(), left.item()) == want


def test_pages_come_and_go(cuda):
    """A server's steps: prompts come, tokens are added, some drafts are taken back, sequences end; no page is ever in two places."""
    rng, batch, width, page, pool = random.Random(5), 9, 12, 16, 70
    table, free = torch.full((batch, width), -1, dtype=torch.int32, device=cuda), torch.arange(pool, dtype=torch.int32, device=cuda).flip(0).contiguous()
    counts, lengths = [_i32([pool], cuda), _i32([0], cuda)], [0] * batch
    for step in range(40):
        kept = [rng.choice([n, n, max(0, n - rng.randint(0, 20)), 0]) for n in lengths]
        ktt.paged_release(table, _i32(lengths, cuda), _i32(kept, cuda), free, counts[0], page, counts[1])
        added = [rng.choice([1, 1, 0, rng.randint(0, 90)]) if n + 90 < width * page else 0 for n in kept]
        cu, positions, slots, granted = ktt.paged_reserve(table, _i32(kept, cuda), _i32(added, cuda), free, counts[1], page, sum(added), counts[0])
        lengths = [n + m for n, m in zip(kept, granted.tolist())]
        count = counts[0].item()
        mine = [p for row, n in zip(table.tolist(), lengths) for p in row[:-(-n // page)]]
        assert all(p == -1 for row, n in zip(table.tolist(), lengths) for p in row[-(-n // page):])
        assert sorted(mine + free[:count].tolist()) == list(range(pool))
        rows = [s for s in slots.tolist() if s >= 0]
        assert len(rows) == sum(granted.tolist()) == len(set(rows))


def test_rows_of_a_larger_table(cuda, path):
    """A table that is part of another, wider one: what is beside it stays."""
    whole = torch.full((4, 9), -5, dtype=torch.int32, device=cuda)
    part = whole[1:3, 2:6]
    part.fill_(-1)
    left = _i32([0], cuda)
    ktt.paged_reserve(part, _i32([0, 0], cuda), _i32([20, 64], cuda), _i32([5, 6, 7, 8, 9, 10], cuda), _i32([6], cuda), 16, 84, left)
    assert part.tolist() == [[10, 9, -1, -1], [8, 7, 6, 5]] and left.item() == 0
    ktt.paged_release(part, _i32([20, 64], cuda), _i32([0, 17], cuda), _i32([0] * 6, cuda), _i32([0], cuda), 16, left)
    assert part.tolist() == [[-1, -1, -1, -1], [8, 7, -1, -1]] and left.item() == 1      # (of 10, 9, 6 and 5: a list of 6 is of pages 0 to 5)
    whole[1:3, 2:6] = -5
    assert torch.equal(whole, torch.full_like(whole, -5))


def test_refusals(cuda, path):
    t, n, f, c, o = _i32([[-1, -1]], cuda), _i32([0], cuda), _i32([1, 2], cuda), _i32([2], cuda), _i32([0], cuda)
    for bad, error in (((t.long(), n, n, f, c, 16, 1, o), ValueError), ((t, n.long(), n, f, c, 16, 1, o), ValueError), ((t, n, _i32([0, 0], cuda), f, c, 16, 1, o), ValueError),
                       ((t, n, n, f.long(), c, 16, 1, o), ValueError), ((t, n, n, f, f, 16, 1, o), ValueError), ((t, n, n, f, c, 16, 1, c), ValueError),
                       ((t, n, n, f, c, 16, -1, o), ValueError), ((t, n, n, f, c, 20, 1, o), _lib.UnsupportedAttention), ((t, n, n, f[::2], c, 16, 1, o), None),
                       ((t.t(), n, n, f, c, 16, 1, o), ValueError), ((t.expand(2, 2), *[_i32([0, 0], cuda)] * 2, f, c, 16, 1, o), _lib.UnsupportedAttention),
                       ((t, n, n, f.cpu(), c, 16, 1, o), (RuntimeError, ValueError))):
        if error is None:      # (one element: contiguous whatever its stride)
            ktt.paged_reserve(*bad)
            continue
        with pytest.raises(error):
            ktt.paged_reserve(*bad)
    for bad in ((t, n, n, f, c, 16, c), (t, n, n.long(), f, c, 16, o), (t, n, n, f, c, 17, o)):
        with pytest.raises((ValueError, _lib.UnsupportedAttention)):
            ktt.paged_release(*bad)
