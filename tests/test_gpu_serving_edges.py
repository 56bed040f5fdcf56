"""A server's steps where they are not plain: reservations that run short, sequences cut back inside a page, modes that watch operators,
scores that are equal, bounds that lie on one another."""

import random

import pytest
import torch

import kohaku_tt_b200 as ktt
from kohaku_tt_b200 import _lib
from oracle import paged_oracle as po
from oracle import serving_oracle as so

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    """Through the C++ edge, and through Python's."""
    if request.param == "python":
        monkeypatch.setattr(_lib, "_NATIVE", False)


def _x(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def _i32(x, cuda):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


def _held(contents, bits, value=False):
    """What pages of these bf16 values hold."""
    return contents if bits == 16 else po.pack(contents, value)


def _turned(k, at, cos, sin):
    """Rows [n, Hk, D] by their positions."""
    at = torch.tensor(at, dtype=torch.long)
    return po.turn_fp32(k, cos[at][:, None], sin[at][:, None], False)


def _near(got, want, mag, size):
    """As in the tests of attention over tables of a token's own."""
    e = 2.0 ** -8
    room = e * want.abs() + (e + 2.0 ** -16 + torch.expm1(2 * 2.0 ** -18 * size[..., None])) * (1 + e) * mag + 1e-30
    off = (got.double().cpu() - want).abs()
    assert bool((off <= room).all()), (off - room).max().item()


# ---- rows that a reservation had no room for ----------------------------------------------------

GRANTED = [  # lengths, new rows of each sequence, granted
    ([0, 20, 16, 47], [3, 30, 1, 40], [3, 0, 1, 0]),
    ([5, 15, 31, 0], [1, 1, 1, 1], [1, 0, 0, 1]),
    ([5, 15, 31, 0], [1, 1, 1, 1], [0, 0, 0, 0]),
    ([100, 90, 3, 0], [70, 0, 33, 16], [12, 5, 99, -4]),     # some of a sequence's, more than there are, fewer than none
    ([127, 128, 126, -3], [4, 4, 4, 4], [4, 4, 1, 4]),       # past the table's end
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lengths,new,granted", GRANTED)
@pytest.mark.parametrize("many", [False, True])
def test_append_of_granted_rows(cuda, path, bits, d, lengths, new, granted, many):
    """The first granted[b] rows of each sequence are in the cache, in the bounds and in the new lengths; queries turn all. Packed, and where
    all have as many rows dense; of 4 and of 40 sequences (whose rows are looked up in another way)."""
    hk, h, page, wide = 2, 4, 16, 8
    if many:
        lengths, new, granted = lengths * 10, new * 10, granted * 10
    batch, total = len(lengths), sum(new)
    table = torch.randperm(batch * wide, generator=torch.Generator().manual_seed(1)).view(batch, wide).to(torch.int32)
    table[1, -1] = -1
    k, v, q = _x(total, hk, d, seed=2), _x(total, hk, d, seed=3), _x(total, h, d, seed=4)
    cos, sin = ktt.rotary_table(wide * page + 99, d, device=cuda)
    starts = [min(max(n, 0), wide * page) for n in lengths]
    places = [n + i for n, m in zip(starts, new) for i in range(m)]
    for positions in (None, torch.tensor(places, dtype=torch.int32, device=cuda) // 2):
        turned = _turned(k, places if positions is None else [x // 2 for x in places], cos.cpu(), sin.cpu())
        kc, vc = _x(batch * wide, hk, page, d, seed=5), _x(batch * wide, hk, page, d, seed=6)
        kp, vp = (_held(x, bits, value).to(cuda) for x, value in ((kc, False), (vc, True)))
        td, lens = table.to(cuda), _i32(lengths, cuda)
        plain = torch.full((batch * wide, hk, 2, d), 7.0, dtype=torch.bfloat16)
        bounds = so.bounds(_held(kc, bits), table, lengths, plain)
        after = so.append(kc, table, lengths, turned.split(new), granted)
        assert after == so.append(vc, table, lengths, v.split(new), granted)
        want_bounds = so.bounds(_held(kc, bits), table, after, plain)
        want_q = _turned(q, places if positions is None else [x // 2 for x in places], cos.cpu(), sin.cpu())
        forms = [(k, v, q, positions, dict(cu_seq=_i32([sum(new[:i]) for i in range(batch + 1)], cuda)))]
        if len(set(new)) == 1:
            dense = [x.view(batch, new[0], -1, d).transpose(1, 2) for x in (k, v, q)]
            forms.append((*dense, None if positions is None else positions.view(batch, -1), {}))
        for kn, vn, qn, pos, kw in forms:
            for edges in (None, bounds.to(cuda)):
                into, out = (kp.clone(), vp.clone()), _i32([-1] * batch, cuda)
                got = ktt.paged_append(kn.to(cuda), vn.to(cuda), *into, td, lens, cos, sin, q=qn.to(cuda), lengths_out=out, positions=pos, bounds=edges,
                                       granted=_i32(granted, cuda), **kw)
                assert out.tolist() == after
                assert torch.equal(into[0].cpu(), _held(kc, bits)) and torch.equal(into[1].cpu(), _held(vc, bits, True))
                assert edges is None or torch.equal(edges.cpu(), want_bounds)
                assert torch.equal((got if kw else got.transpose(1, 2).reshape(total, h, d)).cpu(), want_q)


@pytest.mark.parametrize("bits", [16, 4])
def test_steps_that_run_short(cuda, path, bits):
    """Steps of a server whose list of free pages runs short: what was refused is asked for again, pages come back as sequences end. Tables,
    lengths, pages, bounds and outputs are the definitions'."""
    d, h, hk, page, wide, pool, top, batch = 64, 4, 2, 16, 10, 17, 3, 4
    rng = random.Random(3)
    kp, vp = ktt.paged_cache(pool, hk, page, d, bits=bits, device=cuda)
    kc, vc = torch.zeros((pool, hk, page, d), dtype=torch.bfloat16), torch.zeros((pool, hk, page, d), dtype=torch.bfloat16)
    table, free, count = [[-1] * wide for _ in range(batch)], list(range(pool)), pool
    td, fd, left, now = _i32(table, cuda), _i32(free, cuda), _i32([0], cuda), _i32([pool], cuda)
    lens, after, have = _i32([0] * batch, cuda), _i32([0] * batch, cuda), [0] * batch
    bounds = ktt.paged_bounds(kp, td, lens)
    cos, sin = ktt.rotary_table(wide * page, d, device=cuda)
    refused, waiting, later = 0, [False] * batch, 0
    ask = [rng.randint(20, 60) for _ in range(batch)]
    for step in range(24):
        total = sum(ask)
        q, k, v = _x(total, h, d, seed=step), _x(total, hk, d, seed=step + 100), _x(total, hk, d, seed=step + 200)
        cu, at, slots, granted = ktt.paged_reserve(td, lens, _i32(ask, cuda), fd, now, page, total, left)
        turned = ktt.paged_append(k.to(cuda), v.to(cuda), kp, vp, td, lens, cos, sin, q=q.to(cuda), cu_seq=cu, lengths_out=after, bounds=bounds, granted=granted)
        chosen, keys = ktt.paged_select(turned, bounds, td, after, page, top, cu_seq_q=cu)
        out = ktt.sdpa_paged(turned, kp, vp, chosen, keys)
        table, _, places, want_slots, some, count = so.reserve(table, have, ask, free, count, page, total)
        assert td.tolist() == table and granted.tolist() == some and left.item() == count and slots.tolist() == want_slots and at.tolist() == places
        names = torch.tensor(table, dtype=torch.int32)
        so.append(vc, names, have, v.split(ask), some)
        have = so.append(kc, names, have, _turned(k, places, cos.cpu(), sin.cpu()).split(ask), some)
        assert after.tolist() == have
        assert torch.equal(kp.cpu(), _held(kc, bits)) and torch.equal(vp.cpu(), _held(vc, bits, True))
        want = so.bounds(_held(kc, bits), names, have, bounds.cpu())
        assert torch.equal(bounds.cpu(), want)
        rows = [r for r, b in enumerate(b for b in range(batch) for _ in range(ask[b])) if some[b] == ask[b]]
        owners = so.tokens(ask, have, wide * page)
        want, want_keys = so.select(turned.cpu()[rows], bounds.cpu(), names, [owners[r] for r in rows], page, top, 1, 1)
        assert torch.equal(chosen.cpu()[rows], want) and torch.equal(keys.cpu()[rows], want_keys)
        _near(out[rows], *so.attend(turned.cpu()[rows], kp.cpu(), vp.cpu(), want, want_keys, d ** -0.5))
        refused += sum(x != y for x, y in zip(ask, some))
        later += sum(was and x == y for was, x, y in zip(waiting, ask, some))
        waiting = [x != y for x, y in zip(ask, some)]
        # Some sequences end; what was refused is asked for again.
        kept = [0 if n > wide * page - 70 or rng.random() < 0.1 else n for n in have]
        ktt.paged_release(td, after, _i32(kept, cuda), fd, left, page, now)
        table, free, count = so.release(table, have, kept, free, count, page)
        assert td.tolist() == table and now.item() == count and fd.tolist()[:count] == free[:count]
        ask = [x if x != y else (rng.randint(1, 60) if n == 0 else rng.choice([1, 1, 20])) for x, y, n in zip(ask, some, kept)]
        have = kept
        lens.copy_(_i32(have, cuda))
    assert refused > 5 and later > 2


def test_granted_refusals(cuda, path):
    row, kp = torch.zeros((1, 2, 1, 64), dtype=torch.bfloat16, device=cuda), torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16, device=cuda)
    table, n, out = _i32([[0, 1]], cuda), _i32([3], cuda), _i32([0], cuda)
    for bad in (n.long(), _i32([1, 1], cuda), _i32([[1]], cuda), out):      # (out: what the launch writes)
        with pytest.raises(ValueError):
            ktt.paged_append(row, row, kp, kp, table, n, lengths_out=out, granted=bad)
    with pytest.raises((RuntimeError, ValueError)):
        ktt.paged_append(row, row, kp, kp, table, n, granted=torch.ones(1, dtype=torch.int32))


def test_granted_compiled_and_captured(cuda):
    """The append of granted rows in a compiled graph and in a captured one, as the eager call."""
    d, hk, page, wide, batch = 64, 2, 16, 4, 3
    table, lens, granted = _i32([[0, 1, 2, 3], [4, 5, -1, -1], [6, -1, -1, -1]], cuda), _i32([20, 30, 0], cuda), _i32([1, 0, 1], cuda)
    rows = [_x(batch, n, 1, d, seed=n).to(cuda) for n in (hk, hk, 4)]
    cos, sin = ktt.rotary_table(wide * page, d, device=cuda)

    def fresh():
        return (*(_x(8, hk, page, d, seed=s).to(cuda) for s in (7, 8)), torch.zeros((8, hk, 2, d), dtype=torch.bfloat16, device=cuda), _i32([-1] * batch, cuda))

    def step(k, v, q, kp, vp, bounds, out):
        return ktt.paged_append(k, v, kp, vp, table, lens, cos, sin, q=q, lengths_out=out, bounds=bounds, granted=granted)

    first, second, third = fresh(), fresh(), fresh()
    want = step(*rows, *first)
    assert first[3].tolist() == [21, 30, 1]
    got = torch.compile(step, fullgraph=True)(*rows, *second)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*rows, *third)
    graph.replay()
    assert torch.equal(got, want) and torch.equal(captured, want)
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


# ---- sequences cut back inside a page -----------------------------------------------------------

def _equal(got, want):
    assert torch.equal(got.cpu().float().nan_to_num(7777.0), want.float().nan_to_num(7777.0))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 48)])
@pytest.mark.parametrize("how", ["release", "since"])
@pytest.mark.parametrize("odd", [False, True])
def test_bounds_of_a_cut_back_cache(cuda, path, bits, d, page, how, odd):
    """Drafts that were not taken leave nothing in the bounds, not even NaN: they are those made of the whole cache, after the cut and after
    the appends behind it, of one row and of several, and so are the selections."""
    hk, h, wide, batch, top = 2, 4, 7, 6, 3
    lengths = [3 * page + 5, 2 * page, page + 1, 7, 5 * page - 1, 0]
    drafts = 6
    table = torch.randperm(batch * wide, generator=torch.Generator().manual_seed(1)).view(batch, wide).to(torch.int32)
    kc = _x(batch * wide, hk, page, d, seed=2)
    full = torch.full((batch * wide, hk, 2, d), 7.0, dtype=torch.bfloat16)
    td, kp = table.to(cuda), _held(kc, bits).to(cuda)
    vp, bounds = kp.clone(), so.bounds(_held(kc, bits), table, lengths, full).to(cuda)
    free, left, count = _i32([0] * (batch * wide), cuda), _i32([0], cuda), _i32([0], cuda)

    def append(k, have, n):
        """k: [batch * n, hk, d]."""
        after = _i32([0] * batch, cuda)
        rows = k.view(batch, n, hk, d).transpose(1, 2).to(cuda)
        ktt.paged_append(rows, rows, kp, vp, td, _i32(have, cuda), lengths_out=after, bounds=bounds)
        got = so.append(kc, table, have, k.split(n), [n] * batch)
        assert after.tolist() == got and (odd or torch.equal(kp.cpu(), _held(kc, bits)))
        _equal(bounds, so.bounds(kp.cpu(), table, got, bounds.cpu()))
        return got

    bad = 0
    have = lengths
    for step, taken in enumerate(([0, 1, 2, 6, 5, 0], [9, -1, 6, 0, 3, 6], [6] * 6, [3, 0, 0, 1, 1, 5])):
        k = _x(batch * drafts, hk, d, seed=10 + step) * 4
        if odd:
            k.view(batch, drafts, hk, d)[:, -1, :, 5::7] = float("nan")
            k.view(batch, drafts, hk, d)[:, -2, 0, 3] = float("inf")
        after = append(k, have, drafts)
        kept = [n if t < 0 else min(n + t, a) for n, t, a in zip(have, taken, after)]
        kept = [n - 3 if i == 1 and step == 2 and n > 3 else n for i, n in enumerate(kept)]      # a prompt cut back too
        asked = [k + 5 if k == a else k for k, a in zip(kept, after)]                            # (past the length: it goes on)
        before, held = bounds.cpu(), table.clone()
        if how == "release":
            ktt.paged_release(td, _i32(after, cuda), _i32(asked, cuda), free, count, page, left, k_pages=kp, bounds=bounds)
            td.copy_(table)      # (the pages again, for the steps to come)
        else:
            ktt.paged_bounds(kp, td, _i32(kept, cuda), bounds=bounds, since=_i32(kept, cuda) // page * page)
        assert torch.equal(table, held)
        _equal(bounds, so.bounds(kp.cpu(), table, kept, before))
        bad += int(before.isnan().sum()) > int(bounds.isnan().sum())
        # (and of pages that are not cut nothing moved)
        cut = {int(table[b, n // page]) for b, (n, a) in enumerate(zip(kept, after)) if n % page and n < a}
        others = [i for i in range(batch * wide) if i not in cut]
        _equal(bounds[others], before[others])
        have = append(_x(batch, hk, d, seed=50 + step), kept, 1)
        q = _x(batch, h, d, seed=70 + step)
        chosen, keys = ktt.paged_select(q[:, :, None].to(cuda), bounds, td, _i32(have, cuda), page, top)
        want, want_keys = so.select(q, bounds.cpu(), table, so.tokens([1] * batch, have, wide * page), page, top, 1, 1)
        assert torch.equal(chosen.cpu(), want) and torch.equal(keys.cpu(), want_keys)
    assert bool(bad) == odd


def test_release_with_bounds_refusals(cuda, path):
    kp = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16, device=cuda)
    bounds = torch.zeros((4, 2, 2, 64), dtype=torch.bfloat16, device=cuda)
    t, n, f, c, o = _i32([[0, 1]], cuda), _i32([20], cuda), _i32([0] * 4, cuda), _i32([0], cuda), _i32([0], cuda)
    for kw, error in ((dict(k_pages=kp), ValueError), (dict(bounds=bounds), ValueError), (dict(k_pages=kp, bounds=bounds[:3]), ValueError), (dict(k_pages=kp, bounds=bounds.float()), ValueError),
                      (dict(k_pages=torch.zeros((4, 2, 32, 64), dtype=torch.bfloat16, device=cuda), bounds=bounds), ValueError),
                      (dict(k_pages=kp, bounds=bounds[:1].expand(4, 2, 2, 64)), _lib.UnsupportedAttention)):
        with pytest.raises(error):
            ktt.paged_release(t, n, _i32([3], cuda), f, c, 16, o, **kw)
    torch.cuda.synchronize()
    assert t.tolist() == [[0, 1]] and o.item() == 0      # (nothing was launched)


def test_release_with_bounds_compiled_and_captured(cuda):
    kp, table, n, kept = _x(8, 2, 16, 64, seed=1).to(cuda), _i32([[0, 1, 2], [3, 4, -1]], cuda), _i32([40, 20], cuda), _i32([21, 20], cuda)
    base = ktt.paged_bounds(kp, table, n)

    def fresh():
        return table.clone(), base.clone(), _i32([9] * 8, cuda), _i32([-1], cuda)

    def step(table, bounds, free, left):
        ktt.paged_release(table, n, kept, free, _c, 16, left, k_pages=kp, bounds=bounds)
        return left + 0

    _c = _i32([0], cuda)
    first, second, third = fresh(), fresh(), fresh()
    step(*first)
    assert first[3].item() == 1 and first[0].tolist() == [[0, 1, -1], [3, 4, -1]] and not torch.equal(first[1], base)
    torch.compile(step, fullgraph=True)(*second)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*third)
    graph.replay()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


# ---- modes that watch operators -----------------------------------------------------------------

def test_a_mode_sees_the_operators(cuda):
    """Under a dispatch mode each entry is its operator, with the eager call's results; a rotation has its gradients there, and theirs."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    b, h, hk, d, page, wide, t = 3, 8, 2, 64, 16, 4, 9
    q, k, v = _x(t, h, d, seed=1).to(cuda), _x(t, hk, d, seed=2).to(cuda), _x(t, hk, d, seed=3).to(cuda)
    cos, sin = ktt.rotary_table(wide * page, d, device=cuda)
    axes, offsets = tuple(i % 3 for i in range(d // 2)), [0, 4, 4, 9]

    def step():
        kp, vp = ktt.paged_cache(12, hk, page, d, device=cuda)
        table, lens, after = torch.full((b, wide), -1, dtype=torch.int32, device=cuda), _i32([0] * b, cuda), _i32([0] * b, cuda)
        free, count, left = torch.arange(12, dtype=torch.int32, device=cuda), _i32([12], cuda), _i32([0], cuda)
        bounds = torch.zeros((12, hk, 2, d), dtype=torch.bfloat16, device=cuda)
        cu, at, slots, granted = ktt.paged_reserve(table, lens, _i32([4, 0, 5], cuda), free, count, page, t, left)
        turned = ktt.paged_append(k, v, kp, vp, table, lens, cos, sin, q=q, cu_seq=offsets, lengths_out=after, positions=at.expand(3, t), axes=axes, bounds=bounds, granted=granted)
        ktt.paged_append(k, v, kp, vp, table, after, cu_seq=cu)
        again = ktt.paged_bounds(kp, table, after)
        chosen, keys = ktt.paged_select(turned, bounds, table, after, page, 2, cu_seq_q=offsets)
        outs = ktt.sdpa_paged(turned, kp, vp, chosen, keys), ktt.sdpa_paged(turned, kp, vp, table, after, cu_seq_q=offsets), *ktt.paged_read(kp, vp, table, after)
        ktt.paged_release(table, after, _i32([0, 0, 2], cuda), free, left, page, count, k_pages=kp, bounds=bounds)
        return cu, at, slots, granted, turned, again, chosen, keys, *outs, table, free, count, left, after, bounds, kp, vp

    def gradients():
        x, y, w = (z.clone().requires_grad_() for z in (q, k, q))
        a, c = ktt.rotary(x, y, cos, sin, positions=torch.arange(t, device=cuda).expand(3, t), axes=axes)
        (g,) = torch.autograd.grad((a * w).sum() + c.sum(), x, create_graph=True)
        return a, c, g, torch.autograd.grad(g.sum(), w)[0], ktt.rotary(x, None, cos, sin, interleaved=True)[0]

    want = step() + gradients()
    with Seen() as seen:
        got = step() + gradients()
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    for name in ("_paged_reserve", "_paged_append_at", "_paged_append", "_paged_select", "_sdpa_paged_chosen", "_sdpa_paged", "_paged_bounds", "_paged_read", "_paged_release", "_rotary",
                 "_rotary_axes"):
        assert f"ktt_b200.{name}.default" in seen.names, name
    with Seen(), pytest.raises(ValueError, match="longest"):
        ktt.sdpa_paged(q, *ktt.paged_cache(2, hk, page, d, device=cuda), _i32([[0], [1], [1]], cuda), _i32([1, 1, 1], cuda), cu_seq_q=offsets, max_q=2)


# ---- bounds that lie on one another -------------------------------------------------------------

def test_written_bounds_on_one_another(cuda, path):
    """Refused where they are written, by strides against each other; read they may be."""
    kp, table, n = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16, device=cuda), _i32([[0, 1, 2, 3]], cuda), _i32([50], cuda)
    row, q = torch.zeros((1, 2, 1, 64), dtype=torch.bfloat16, device=cuda), torch.ones((1, 4, 1, 64), dtype=torch.bfloat16, device=cuda)
    memory = torch.zeros(4096, dtype=torch.bfloat16, device=cuda)
    for strides in ((64, 64, 64), (128, 64, 64), (64, 128, 64), (256, 64, 64), (64, 256, 128)):
        bad = memory.as_strided((4, 2, 2, 64), (*strides, 1))
        for call in (lambda: ktt.paged_bounds(kp, table, n, bounds=bad), lambda: ktt.paged_append(row, row, kp, kp, table, n, bounds=bad),
                     lambda: ktt.paged_release(table, n, n, _i32([0] * 4, cuda), _i32([0], cuda), 16, _i32([0], cuda), k_pages=kp, bounds=bad)):
            with pytest.raises(_lib.UnsupportedAttention, match="on one another"):
                call()
        ktt.paged_select(q, bad, table, n, 16, 2)
    good = memory.as_strided((4, 2, 2, 64), (128, 512, 64, 1))
    assert torch.equal(ktt.paged_bounds(kp + 1, table, n, bounds=good), torch.ones_like(good))


# ---- scores that are equal ----------------------------------------------------------------------

def _first_by_score(q, edge, table, top):
    """Places of the pages between the first and the last, of the largest scores in whole numbers; bounds that are one edge [pages, d], and all values
    multiples of 2^-40."""
    scores = []
    for name in table:
        page = [int(x) for x in (edge[name].double() * 2 ** 40).tolist()]
        scores.append(max(sum(int(a) * b for a, b in zip(row, page)) for row in (q.double() * 2 ** 20).tolist()))
    rest = sorted(range(1, len(table) - 1), key=lambda e: (-scores[e], e))[:top - 2]
    return [int(table[e]) for e in sorted(rest + [0, len(table) - 1])]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("wide", [60, 200, 700, 9000])
def test_equal_scores_in_any_order_of_channels(cuda, d, wide):
    """Pages whose products are the same numbers in other channels, over a factor of almost 2^30, have equal scores and go by place; one that is
    larger by the least product goes first. Against sums in whole numbers."""
    page, top, h = 16, 30, 3
    g = torch.Generator().manual_seed(wide + d)
    q = torch.tensor([1.0, -0.5, 0.25])[:, None].expand(h, d).mul(1.0 + 27 / 128).to(torch.bfloat16)      # a head's channels alike: 8 bits each
    size = 2.0 ** -torch.arange(d).remainder(28) * (1 + torch.randint(0, 128, (d,), generator=g) / 128)
    base = (size * torch.randint(0, 2, (d,), generator=g).mul(2).sub(1)).to(torch.bfloat16)
    edge = torch.stack([base[torch.randperm(d, generator=g)] for _ in range(wide)])
    table = torch.randperm(wide, generator=g).to(torch.int32)
    for some in ([], range(5, wide - 1, 7), [wide // 2], range(1, wide - 1, 2)):
        values = edge.clone()
        least = base.float().abs().min()
        for e in some:      # the least magnitude's sign turned where it is negative, else twice as large: a score that is a little larger
            row = values[table[e].item()]
            i = int((row.float().abs() == least).nonzero()[0])
            row[i] = row[i].abs() if row[i] < 0 else row[i] * 2
        want = _first_by_score(q, values, table.tolist(), top)
        bounds = values[:, None, None].expand(wide, 1, 2, d).contiguous().to(cuda)
        chosen, keys = ktt.paged_select(q.view(1, h, 1, d).to(cuda), bounds, table[None].to(cuda), _i32([wide * page], cuda), page, top)
        assert chosen[0, 0].tolist() == want and keys.item() == top * page
        if not some:
            assert want == table[:top - 1].tolist() + table[-1:].tolist()


# ---- whole numbers past 32 bits -----------------------------------------------------------------

def test_numbers_past_32_bits_are_refused(cuda, path):
    """An argument block would hold what is left of them: pages of 2^32 + 16 keys were pages of 16."""
    far = 2 ** 32
    t, n, f, c, o = _i32([[0, 1]], cuda), _i32([20], cuda), _i32([0] * 4, cuda), _i32([0], cuda), _i32([0], cuda)
    q, bounds = torch.ones((1, 4, 1, 64), dtype=torch.bfloat16, device=cuda), torch.zeros((4, 2, 2, 64), dtype=torch.bfloat16, device=cuda)
    for page in (far + 16, 16 - far):
        for call in (lambda: ktt.paged_reserve(t, n, n, f, c, page, 1, o), lambda: ktt.paged_release(t, n, n, f, c, page, o), lambda: ktt.paged_select(q, bounds, t, n, page, 2)):
            with pytest.raises(_lib.UnsupportedAttention, match="32 bits"):
                call()
    for kw in (dict(top=far + 2), dict(top=2, first=far), dict(top=2, last=far + 1)):
        with pytest.raises(_lib.UnsupportedAttention, match="32 bits"):
            ktt.paged_select(q, bounds, t, n, 16, **kw)
    # Whole numbers of another kind go on being taken.
    import numpy as np
    for page, top in ((np.int64(16), np.int32(2)), (torch.tensor(16), torch.tensor(2))):
        assert ktt.paged_select(q, bounds, t, n, page, top)[0].tolist() == [[[0, 1], [0, 1]]]


# ---- offsets from a list in a compiled graph ----------------------------------------------------

def test_offsets_from_a_list_compiled(cuda):
    """A list of offsets is taken in a compiled graph as it is outside of one, and so are its refusals."""
    h, hk, d, page, t = 4, 2, 64, 16, 9
    q, k, v = (_x(t, n, d, seed=n).to(cuda) for n in (h, hk, hk))
    table, lens, after = _i32([[0, 1], [2, 3], [4, 5]], cuda), _i32([20, 0, 3], cuda), _i32([24, 0, 8], cuda)
    bounds = torch.zeros((6, hk, 2, d), dtype=torch.bfloat16, device=cuda)

    def step(q, k, v, kp, vp, bounds, offsets):
        turned = ktt.paged_append(k, v, kp, vp, table, lens, q=q, cu_seq=offsets, bounds=bounds)
        chosen, keys = ktt.paged_select(turned, bounds, table, after, page, 2, cu_seq_q=offsets)
        return turned, chosen, keys, ktt.sdpa_paged(turned, kp, vp, chosen, keys), ktt.sdpa_paged(turned, kp, vp, table, after, cu_seq_q=offsets)

    def fresh():
        return *(_x(6, hk, page, d, seed=s).to(cuda) for s in (7, 8)), bounds.clone()

    # (By the graph as it was traced: a compiler would write the list's copy in C++, for which a machine that runs these tests need have nothing.)
    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    for offsets in ([0, 4, 4, 9], [0, 0, 5, 9]):
        first, second = fresh(), fresh()
        for x, y in zip((*compiled(q, k, v, *first, offsets), *first), (*step(q, k, v, *second, offsets), *second)):
            assert torch.equal(x, y)
    for bad in ([0, 4, 4], [0, 5, 4, 9], [0, 4, 4, 10]):
        with pytest.raises(Exception, match="offsets must be"):
            torch.compile(step, fullgraph=True, backend="aot_eager")(q, k, v, *fresh(), bad)
