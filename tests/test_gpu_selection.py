"""Bounds of pages, the pages that queries select by them, and attention over tables of a token's own, against float64."""

import pytest
import torch

import kohaku_tt_b200 as ktt
from kohaku_tt_b200 import _lib
from oracle import paged_oracle as po
from oracle import serving_oracle as so

pytestmark = pytest.mark.gpu

BITS = [16, 4]


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    """Through the C++ edge, and through Python's."""
    if request.param == "python":
        monkeypatch.setattr(_lib, "_NATIVE", False)


def _x(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _store(x, bits, value):
    return x if bits == 16 else po.pack(x, value)


def _table(used, wide, pages, seed=0):
    """Pages in no order for the first used[b] entries of each row, -1 behind them."""
    names = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(used), wide), -1, dtype=torch.int32)
    for b, n in enumerate(used):
        for i in range(n):
            table[b, i] = names.pop()
    return table


def _pages(bits, count, hk, page, d, seed, value=False):
    return _store(_x(count, hk, page, d, seed=seed), bits, value)


def _i32(x, cuda):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


def _same(got, want):
    assert torch.equal(got.cpu().float().nan_to_num(7777.0), want.float().nan_to_num(7777.0))


# ---- bounds -------------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("d,hk,page,lengths", [(64, 1, 16, [1]), (128, 2, 16, [0, 1, 15, 16, 17, 40, 64]), (64, 3, 48, [47, 48, 49, 0, 200]), (128, 8, 256, [700, 255, 1]),
                                               (64, 2, 32, [-5, 1000])])
def test_bounds(cuda, path, bits, d, hk, page, lengths):
    wide = 6
    used = [min(max(-(-n // page), 0), wide) for n in lengths]
    count = sum(used) + 2
    kp, table = _pages(bits, count, hk, page, d, 1), _table(used, wide, count)
    if max(used) > 2:
        table[lengths.index(max(lengths)), 1] = count      # no page of the cache
    zero = torch.zeros((count, hk, 2, d), dtype=torch.bfloat16)
    want = so.bounds(kp, table, lengths, zero)
    lens, td, kd = _i32(lengths, cuda), table.to(cuda), kp.to(cuda)
    got = ktt.paged_bounds(kd, td, lens)
    assert got.dtype == torch.bfloat16
    _same(got, want)
    # In place, in parts: a third of the keys, then the rest on top.
    some = [max(n, 0) // 3 for n in lengths]
    into = torch.full_like(got, 9.0)
    assert ktt.paged_bounds(kd, td, _i32(some, cuda), bounds=into) is into
    assert ktt.paged_bounds(kd, td, lens, bounds=into, since=_i32(some, cuda)) is into
    _same(into, so.bounds(kp, table, lengths, torch.full_like(zero, 9.0)))
    # Nothing new: nothing changes. Past the length and below 0: taken as its ends.
    before = into.clone()
    ktt.paged_bounds(kd, td, lens, bounds=into, since=lens + 5)
    assert torch.equal(into, before)
    ktt.paged_bounds(kd, td, lens, bounds=into, since=torch.full_like(lens, -3))
    assert torch.equal(into, before)


def test_bounds_of_odd_values(cuda):
    """A NaN stays, in its channel; infinities are values; what lies behind the length is nothing."""
    kp = _x(3, 2, 16, 64, seed=2)
    kp[0, 0, 3, 5], kp[0, 1, 2, 7], kp[1, 0, 0, 1], kp[1, 0, 4:] = float("nan"), float("inf"), float("-inf"), float("nan")
    table, lengths = torch.tensor([[0, 1, 2]], dtype=torch.int32), [20]
    want = so.bounds(kp, table, lengths, torch.zeros((3, 2, 2, 64), dtype=torch.bfloat16))
    got = ktt.paged_bounds(kp.to(cuda), table.to(cuda), _i32(lengths, cuda))
    _same(got, want)
    assert got.isnan().sum() == 2 and got[0, 0, 0, 5].isnan() and got[0, 1, 1, 7] == float("inf") and got[1, 0, 0, 1] == float("-inf")


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,packed", [([1, 1, 1, 1], False), ([40, 40, 40, 40], False), ([16, 16, 16, 16], False), ([1, 0, 70, 33], True), ([1, 1, 1, 1], True), ([0, 0, 0, 5], True)])
def test_append_keeps_bounds(cuda, path, bits, d, new, packed):
    """As paged_bounds makes them of the pages afterwards, wherever in a page the rows begin; a place without a page takes nothing."""
    hk, page, wide = 3, 16, 8
    for lengths in ([0, 5, 15, 16], [17, 31, 48, 63], [128, 127, 100, 96]):
        used = [min(wide, -(-(n + m) // page)) for n, m in zip(lengths, new)]
        count = sum(used) + 1
        table = _table(used, wide, count, seed=3)
        table[1, -1] = -1
        kp, vp = _pages(bits, count, hk, page, d, 4).to(cuda), _pages(bits, count, hk, page, d, 5, True).to(cuda)
        td, lens, after = table.to(cuda), _i32(lengths, cuda), _i32([0] * 4, cuda)
        bounds = ktt.paged_bounds(kp, td, lens, bounds=torch.full((count, hk, 2, d), 7.0, dtype=torch.bfloat16, device=cuda))
        total = sum(new)
        k, v = _x(total, hk, d, seed=6) * 2, _x(total, hk, d, seed=7)
        cos, sin = ktt.rotary_table(wide * page, 32, device=cuda)
        if packed:
            cu = [0]
            for n in new:
                cu.append(cu[-1] + n)
            pad = torch.full((3, hk, d), float("nan"), dtype=torch.bfloat16)      # rows of no sequence
            kw, rows = dict(cu_seq=_i32(cu, cuda)), [torch.cat([x, pad]).to(cuda) for x in (k, v)]
        else:
            kw, rows = {}, [x.view(4, new[0], hk, d).transpose(1, 2).to(cuda) for x in (k, v)]
        ktt.paged_append(*rows, kp, vp, td, lens, cos, sin, lengths_out=after, bounds=bounds, **kw)
        want = so.bounds(kp.cpu(), table, after.tolist(), torch.full((count, hk, 2, d), 7.0, dtype=torch.bfloat16))
        _same(bounds, want)
        # Pages and lengths are those of an append without bounds.
        kp2, vp2 = _pages(bits, count, hk, page, d, 4).to(cuda), _pages(bits, count, hk, page, d, 5, True).to(cuda)
        ktt.paged_append(*rows, kp2, vp2, td, lens, cos, sin, **kw)
        assert torch.equal(kp.view(torch.uint8), kp2.view(torch.uint8)) and torch.equal(vp.view(torch.uint8), vp2.view(torch.uint8))


# ---- the selection ------------------------------------------------------------------------------

def _selected(cuda, q, bounds, table, lengths, counts, page, top, first, last, packed, tail=0):
    """Both forms of the call against the oracle; returns what the device chose."""
    cap = table.shape[1] * page
    owners = so.tokens(counts, lengths, cap) + [(0, 0)] * tail
    want, want_keys = so.select(q, bounds, table, owners, page, top, first, last)
    bd, td, lens = bounds.to(cuda), table.to(cuda), _i32(lengths, cuda)
    if packed:
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        chosen, keys = ktt.paged_select(q.to(cuda), bd, td, lens, page, top, first=first, last=last, cu_seq_q=_i32(cu, cuda))
    else:
        b, n = len(counts), counts[0]
        rows = q.view(b, n, *q.shape[1:]).transpose(1, 2).to(cuda)
        chosen, keys = ktt.paged_select(rows, bd, td, lens, page, top, first=first, last=last)
    assert chosen.shape == want.shape and chosen.dtype == keys.dtype == torch.int32
    assert torch.equal(keys.cpu(), want_keys) and torch.equal(chosen.cpu(), want)
    return chosen, keys


SELECT = [  # D, H, Hk, page, table width, tokens, lengths, top, first, last
    (128, 16, 2, 16, 100, [1, 1, 1, 1], [1600, 1, 0, 777], 12, 1, 2),
    (64, 14, 2, 16, 40, [3, 3], [500, 40], 9, 0, 1),
    (64, 4, 4, 32, 30, [1, 1, 1], [960, 95, 31], 3, 1, 1),
    (128, 40, 2, 16, 33, [1, 1], [520, 300], 8, 2, 4),           # more than 16 heads to a key head
    (128, 24, 2, 48, 20, [2, 2], [900, 100], 5, 4, 1),           # nothing but the first and the last
    (64, 2, 1, 16, 700, [1], [11111], 100, 1, 1),
    (128, 8, 8, 64, 17, [5, 0, 1, 16], [1000, 3, 64, 16], 6, 1, 1),
    (64, 8, 1, 16, 2300, [1], [36800], 64, 4, 8),
]


@pytest.mark.parametrize("d,h,hk,page,wide,counts,lengths,top,first,last", SELECT)
@pytest.mark.parametrize("packed", [False, True])
def test_select(cuda, path, d, h, hk, page, wide, counts, lengths, top, first, last, packed):
    if not packed and len(set(counts)) > 1:
        counts = [4] * len(counts)
    pages = len(lengths) * wide
    x = _x(pages, hk, 2, d, seed=1).float().sort(dim=2).values.to(torch.bfloat16)
    table = _table([wide] * len(lengths), wide, pages, seed=2)
    tail = 2 if packed else 0
    q = _x(sum(counts) + tail, h, d, seed=3)
    _selected(cuda, q, x, table, lengths, counts, page, top, first, last, packed, tail)


@pytest.mark.parametrize("d,h,hk", [(64, 4, 2), (128, 16, 1)])
def test_equal_and_nearly_equal_scores(cuda, d, h, hk):
    """Ties go to the first page; scores apart by less than fp32 sums are off by are told apart; in tens, in hundreds, and all alike."""
    page, wide, top = 16, 600, 40
    table = _table([wide], wide, wide, seed=2)
    q = _x(1, h, d, seed=3)
    base = _x(1, hk, 2, d, seed=4).float().sort(dim=2).values.to(torch.bfloat16)
    alike = base.expand(wide, hk, 2, d).clone()
    _selected(cuda, q, alike, table, [wide * page], [1], page, top, 1, 1, False)
    # One channel differs by a little: by less than 2^-24 of the sum.
    near = alike.clone()
    near[:, :, :, 0] = (near[:, :, :, 0].float().sign() * 2.0 ** -20 * (1 + torch.arange(wide).remainder(97)[:, None, None] / 128)).to(torch.bfloat16)
    _selected(cuda, q, near, table, [wide * page], [1], page, top, 1, 1, False)
    # Three kinds, far apart.
    kinds = torch.where(torch.arange(wide).remainder(3)[:, None, None, None] == 0, alike, alike * 2)
    kinds = torch.where(torch.arange(wide).remainder(50)[:, None, None, None] == 7, alike * 4, kinds)
    _selected(cuda, q, kinds, table, [wide * page], [1], page, top, 1, 1, False)
    # Few differ from a mass of zeros; queries of zeros.
    few = torch.zeros_like(alike)
    few[::17] = _x(few[::17].shape[0], hk, 2, d, seed=5).float().sort(dim=2).values.to(torch.bfloat16)
    _selected(cuda, q, few, table, [wide * page], [1], page, top, 1, 1, False)
    _selected(cuda, torch.zeros_like(q), few, table, [wide * page], [1], page, top, 1, 1, False)
    # One score far above all others, which then share a bin.
    far = _x(wide, hk, 2, d, seed=6).float().sort(dim=2).values.to(torch.bfloat16)
    far[11] *= 2.0 ** 40
    _selected(cuda, q, far, table, [wide * page], [1], page, top, 1, 1, False)


def test_odd_scores(cuda):
    """NaN counts as infinite, infinities by place, scores past fp32's range by their value; subnormal bounds; missing pages score 0."""
    d, h, hk, page, wide, top = 64, 4, 1, 16, 200, 20
    table = _table([wide], wide, wide, seed=2)
    q, x = _x(1, h, d, seed=3), _x(wide, hk, 2, d, seed=4).float().sort(dim=2).values.to(torch.bfloat16)
    missing = table.clone()
    missing[0, 5:60:3], missing[0, 70] = -1, wide
    _selected(cuda, q, x, missing, [wide * page], [1], page, top, 1, 1, False)
    odd = x.clone()
    odd[3, 0, 0, 1], odd[9, 0, 1, 2], odd[40, 0, 0, 3], odd[77, 0] = float("nan"), float("inf"), float("-inf"), float("nan")
    _selected(cuda, q, odd, table, [wide * page], [1], page, top, 1, 1, False)
    _selected(cuda, (q.float() * 1e30).to(torch.bfloat16), (x.float() * 1e30).to(torch.bfloat16), table, [wide * page], [1], page, top, 1, 1, False)
    _selected(cuda, q, (x.float() * 1e-39).to(torch.bfloat16), table, [wide * page], [1], page, top, 1, 1, False)
    _selected(cuda, (q.float() * 1e-30).to(torch.bfloat16), (x.float() * 1e-20).to(torch.bfloat16), table, [wide * page], [1], page, top, 1, 1, False)
    bad = q.clone()
    bad[0, 2, 7] = float("nan")
    _selected(cuda, bad, x, table, [wide * page], [1], page, top, 1, 1, False)


def test_scores_that_do_not_fit_shared_memory(cuda):
    page, wide, top, d = 16, 60000, 50, 64
    x = _x(wide, 1, 2, d, seed=1).float().sort(dim=2).values.to(torch.bfloat16)
    table = torch.arange(wide, dtype=torch.int32)[None]
    q = _x(2, 2, d, seed=2)
    got, keys = ktt.paged_select(q.view(1, 2, 2, d).transpose(1, 2).to(cuda), x.to(cuda), table.to(cuda), _i32([wide * page], cuda), page, top)
    b = x.double()
    for t in range(2):
        score = torch.stack([torch.maximum(y * b[:, 0, 0], y * b[:, 0, 1]).sum(-1) for y in q[t].double()]).amax(0)
        best = torch.sort(score[1:-1], descending=True, stable=True).indices[:top - 2] + 1
        assert got[t, 0].tolist() == sorted(best.tolist() + [0, wide - 1]) and keys[t, 0] == top * page - (1 - t)


def test_many_tokens_in_several_launches(cuda):
    """More scores than are kept at a time: tokens of a later launch are as those of the first."""
    d, h, hk, page, wide, top, t = 64, 32, 32, 16, 9000, 5, 80
    x = _x(wide, hk, 2, d, seed=1).float().sort(dim=2).values.to(torch.bfloat16).to(cuda)
    table = torch.arange(wide, dtype=torch.int32, device=cuda).expand(t, wide).contiguous()
    q = _x(1, h, 1, d, seed=2).to(cuda).expand(t, h, 1, d).contiguous()
    lens = torch.full((t,), wide * page, dtype=torch.int32, device=cuda)
    got, keys = ktt.paged_select(q, x, table, lens, page, top)
    one, _ = ktt.paged_select(q[:1], x, table[:1], lens[:1], page, top)
    assert torch.equal(got, one.expand_as(got)) and bool((keys == top * page).all())


@pytest.mark.parametrize("d,wide", [(64, 512), (64, 513), (64, 1024), (64, 1025), (64, 2049), (64, 4096), (64, 4097), (128, 512), (128, 1025), (128, 2048), (128, 2049), (128, 4096), (128, 4100), (128, 8192), (128, 8193)])
def test_widths(cuda, d, wide):
    """Tables about as wide as each way of holding the scores has room for: far apart, two thirds alike, all alike."""
    page, top, h, hk = 16, 70, 4, 1
    table = _table([wide], wide, wide, seed=2)
    q = _x(2, h, d, seed=3)
    x = _x(wide, hk, 2, d, seed=1).float().sort(dim=2).values.to(torch.bfloat16)
    alike = x[:1].expand(wide, hk, 2, d).clone()
    most = torch.where(torch.arange(wide).remainder(3)[:, None, None, None] == 0, x, alike)
    for bounds in (x, most, alike):
        for lengths in ([wide * page], [wide * page - 17 * page - 3]):
            _selected(cuda, q, bounds, table, lengths, [2], page, top, 2, 3, False)


def test_tensors_that_are_no_bounds(cuda):
    """Values of any kind, in no order: pages of the table, each once, in its order, the first and the last among them."""
    page, top, h, hk = 16, 40, 8, 2
    for d, wide in ((64, 300), (128, 2000), (64, 5000)):
        g = torch.Generator().manual_seed(wide)
        table = _table([wide], wide, wide, seed=2)
        place = torch.empty(wide, dtype=torch.long)
        place[table[0].long()] = torch.arange(wide)
        for kind in range(4):
            x = torch.randint(-2 ** 15, 2 ** 15, (wide, hk, 2, d), generator=g, dtype=torch.int16).view(torch.bfloat16)
            if kind == 1:       # large ones the wrong way round
                x = torch.stack([torch.full((wide, hk, d), 3e38), torch.full((wide, hk, d), -3e38)], dim=2).to(torch.bfloat16)
            if kind == 2:
                x = _x(wide, hk, 2, d, seed=4).float().sort(dim=2, descending=True).values.to(torch.bfloat16)
            if kind == 3:       # some of them the wrong way round
                x[::7] = torch.tensor([3e38, -3e38], dtype=torch.bfloat16)[None, None, :, None]
                x[1::7], x[2::7] = 1.0, float("-inf")
            chosen, keys = ktt.paged_select(_x(1, h, 1, d, seed=3).to(cuda), x.to(cuda), table.to(cuda), _i32([wide * page], cuda), page, top)
            assert bool((keys == top * page).all())
            for row in chosen.cpu()[0]:
                at = place[row.long()]
                assert bool((at[1:] > at[:-1]).all()) and at[0] == 0 and at[-1] == wide - 1


def test_no_tokens(cuda, path):
    d, h, hk, page = 64, 4, 2, 16
    kp = _x(4, hk, page, d, seed=1).to(cuda)
    bounds, table, lens = torch.zeros((4, hk, 2, d), dtype=torch.bfloat16, device=cuda), _table([2, 2], 2, 4).to(cuda), _i32([20, 0], cuda)
    for q, kw in ((_x(0, h, d).to(cuda), dict(cu_seq_q=_i32([0, 0, 0], cuda))), (_x(2, h, 0, d).to(cuda), {})):
        chosen, keys = ktt.paged_select(q, bounds, table, lens, page, 3, **kw)
        assert chosen.shape == (0, hk, 3) and keys.shape == (0, hk)
        assert ktt.sdpa_paged(q, kp, kp, chosen, keys).shape == q.shape


def test_layouts(cuda, path):
    """Queries as head views and at odd places, bounds in another order and in parts of a larger tensor, part of a wider table: the same."""
    d, h, hk, page, wide, b, top = 64, 8, 2, 16, 50, 3, 9
    x = _x(b * wide, hk, 2, d, seed=1).float().sort(dim=2).values.to(torch.bfloat16).to(cuda)
    table, lens = _table([wide] * b, wide, b * wide, seed=2).to(cuda), _i32([800, 333, 640], cuda)
    q = _x(b, h, 2, d, seed=3).to(cuda)
    want = ktt.paged_select(q, x, table, lens, page, top)
    flat = torch.empty(b * 2 * h * d + 3, dtype=torch.bfloat16, device=cuda)
    odd = flat[3:].view(b, h, 2, d)
    odd.copy_(q)
    turned = x.transpose(1, 2).contiguous().transpose(1, 2)
    larger = torch.zeros((b * wide, hk + 1, 3, d + 8), dtype=torch.bfloat16, device=cuda)
    part = larger[:, 1:, :2, 8:]
    part.copy_(x)
    wider = torch.zeros((b, wide + 5), dtype=torch.int32, device=cuda)
    wider[:, :wide] = table
    views = q.transpose(1, 2).reshape(b, 2, h * d).view(b, 2, h, d).transpose(1, 2)
    for args in ((odd, x, table), (views, x, table), (q, turned, table), (q, part, table), (q, x, wider[:, :wide])):
        got = ktt.paged_select(*args, lens, page, top)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- attention over tables of a token's own -----------------------------------------------------

def _near(got, want, mag, size):
    """bf16 weights (half a step, 2^-8, of each p |v|) and a bf16 result (2^-8 of it); fp32 sums: 2^-16 of the
    terms. Over 4 bits it is p step that is rounded, before it multiplies code - 8, which `mag` has. Logits: fp32 products,
    2^-18 of sum |q| |k|."""
    e = 2.0 ** -8
    room = e * want.abs() + (e + 2.0 ** -16 + torch.expm1(2 * 2.0 ** -18 * size[..., None])) * (1 + e) * mag + 1e-30
    off = (got.double().cpu() - want).abs()
    assert bool((off <= room).all()), ((off - room).max().item(), off.max().item())


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("d,h,hk,page,top,tokens", [(64, 14, 2, 16, 9, 3), (128, 16, 2, 16, 4, 5), (128, 8, 8, 64, 3, 2), (64, 40, 2, 48, 5, 1), (128, 24, 2, 16, 70, 2),
                                                    (64, 2, 2, 16, 1, 700), (128, 3, 1, 32, 2, 600)])
def test_attention_over_own_tables(cuda, path, bits, d, h, hk, page, top, tokens):
    """Lengths from none to all, an entry that is no page, dense and packed queries."""
    count = 60
    kp, vp = _pages(bits, count, hk, page, d, 1), _pages(bits, count, hk, page, d, 2, True)
    g = torch.Generator().manual_seed(3)
    chosen = torch.randint(0, count, (tokens, hk, top), generator=g).to(torch.int32)
    keys = torch.randint(0, top * page + 1, (tokens, hk), generator=g).to(torch.int32)
    keys[0, 0], keys[-1, -1] = 0, top * page + 9
    if top > 2:
        chosen[0, -1, 1], chosen[-1, 0, 0] = -1, count
    q = _x(tokens, h, d, seed=4)
    some = list(range(tokens)) if tokens < 10 else [0, 1, tokens // 2, tokens - 2, tokens - 1]
    want = so.attend(q[some], kp, vp, chosen[some], keys[some], d ** -0.5)
    args = (kp.to(cuda), vp.to(cuda), chosen.to(cuda), keys.to(cuda))
    out = ktt.sdpa_paged(q.to(cuda), *args)
    assert out.shape == q.shape and out.dtype == q.dtype
    _near(out[some], *want)
    assert bool((out[0, :h // hk] == 0).all())
    dense = ktt.sdpa_paged(q.transpose(0, 1)[None].to(cuda), *args)
    assert torch.equal(dense[0].transpose(0, 1), out)
    each = ktt.sdpa_paged(q[:, :, None].to(cuda), *args)
    assert torch.equal(each[:, :, 0], out)
    want = so.attend(q[some], kp, vp, chosen[some], keys[some].clamp(max=page), 0.3)
    _near(ktt.sdpa_paged(q.to(cuda), *args, scale=0.3, max_k=page)[some], *want)


@pytest.mark.parametrize("bits", BITS)
def test_all_pages_are_attention_over_all(cuda, bits):
    """With room for all pages the selection is the sequence's own table, and the result that of sdpa_paged, to the rounding."""
    d, h, hk, page, lengths = 64, 8, 2, 16, [100, 33, 1]
    kp, vp = _pages(bits, 30, hk, page, d, 1).to(cuda), _pages(bits, 30, hk, page, d, 2, True).to(cuda)
    table, lens, q = _table([7, 3, 1], 10, 30).to(cuda), _i32(lengths, cuda), _x(3, h, 1, d, seed=3).to(cuda)
    chosen, keys = ktt.paged_select(q, ktt.paged_bounds(kp, table, lens), table, lens, page, 10)
    assert torch.equal(chosen, table[:, None].expand(3, hk, 10)) and torch.equal(keys, lens[:, None].expand(3, hk))
    got, want = ktt.sdpa_paged(q, kp, vp, chosen, keys), ktt.sdpa_paged(q, kp, vp, table, lens)
    assert torch.equal(got, want)


def test_more_pairs_than_a_scan_has_room_for(cuda):
    """Long tables of more pairs of token and head than one launch scans: as those of few."""
    d, h, hk, page, top, tokens = 64, 4, 4, 16, 140, 400
    kp, vp = _pages(16, 200, hk, page, d, 1).to(cuda), _pages(16, 200, hk, page, d, 2, True).to(cuda)
    g = torch.Generator().manual_seed(3)
    chosen = torch.randint(0, 200, (tokens, hk, top), generator=g).to(torch.int32)
    keys = torch.randint(1, top * page + 1, (tokens, hk), generator=g).to(torch.int32)
    q = _x(tokens, h, d, seed=4)
    some = [0, 127, 128, 129, 255, 256, 399]
    out = ktt.sdpa_paged(q.to(cuda), kp, vp, chosen.to(cuda), keys.to(cuda))
    _near(out[some], *so.attend(q[some], kp.cpu(), vp.cpu(), chosen[some], keys[some], d ** -0.5))


def test_refusals(cuda, path):
    d, page = 64, 16
    kp = torch.zeros((4, 2, page, d), dtype=torch.bfloat16, device=cuda)
    bounds, table, n = torch.zeros((4, 2, 2, d), dtype=torch.bfloat16, device=cuda), torch.zeros((1, 4), dtype=torch.int32, device=cuda), _i32([3], cuda)
    q = torch.zeros((1, 4, 1, d), dtype=torch.bfloat16, device=cuda)
    for bad in ((q.float(), bounds, table, n, page, 4), (q[..., :32], bounds, table, n, page, 4), (q, bounds.float(), table, n, page, 4), (q, bounds[:, :, :1], table, n, page, 4),
                (q, bounds, table.long(), n, page, 4), (q, bounds, table, n.long(), page, 4), (q, bounds, table, _i32([3, 3], cuda), page, 4), (q[0], bounds, table, n, page, 4),
                (torch.cat([q, q]), bounds, table, n, page, 4)):
        with pytest.raises(ValueError):
            ktt.paged_select(*bad)
    for bad in ((page, 1), (page, 4, 4, 1), (page, 4, -1, 1), (page, 4, 0, 0), (17, 4), (page, -3)):
        with pytest.raises((ValueError, _lib.UnsupportedAttention)):
            ktt.paged_select(q, bounds, table, n, *bad)
    with pytest.raises(_lib.UnsupportedAttention):
        ktt.paged_select(q[:, :3], bounds, table, n, page, 4)
    for bad in (dict(bounds=bounds.float()), dict(bounds=bounds[:3]), dict(bounds=bounds, since=n.long()), dict(bounds=bounds, since=_i32([1, 2], cuda))):
        with pytest.raises(ValueError):
            ktt.paged_bounds(kp, table, n, **bad)
    row = torch.zeros((1, 2, 1, d), dtype=torch.bfloat16, device=cuda)
    for bad in (bounds[:1].expand(4, 2, 2, d), bounds[:, :1].expand(4, 2, 2, d), bounds[:, :, :1].expand(4, 2, 2, d)):      # that lie on one another
        with pytest.raises(_lib.UnsupportedAttention):
            ktt.paged_bounds(kp, table, n, bounds=bad)
        with pytest.raises(_lib.UnsupportedAttention):
            ktt.paged_append(row, row, kp, kp, table, n, bounds=bad)
    chosen, keys = torch.zeros((1, 2, 3), dtype=torch.int32, device=cuda), torch.zeros((1, 2), dtype=torch.int32, device=cuda)
    for bad in ((q, kp, kp, chosen.long(), keys), (q, kp, kp, chosen, keys.long()), (q, kp, kp, chosen, keys[0]), (q, kp, kp, chosen[:, :1], keys[:, :1]),
                (torch.cat([q, q]), kp, kp, chosen, keys), (q[0, 0], kp, kp, chosen, keys)):
        with pytest.raises(ValueError):
            ktt.sdpa_paged(*bad)
    with pytest.raises(ValueError):
        ktt.sdpa_paged(q[0].transpose(0, 1), kp, kp, chosen, keys, cu_seq_q=[0, 1])
