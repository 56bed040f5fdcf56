"""The paged cache: the append, reading back, and attention over pages of bf16 and of 4 bits, against float64."""

import pytest
import torch

import kohaku_tt_b200 as ktt
from kohaku_tt_b200 import _lib
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu

BITS = [16, 4]


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


def _poison(pages, table, lengths, page_size):
    """NaN wherever no sequence has a key: unused pages, and rows behind a sequence's last."""
    live = torch.zeros(pages.shape[0], page_size, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for j in range(n):
            p = int(table[b, j // page_size])
            if 0 <= p < pages.shape[0]:
                live[p, j % page_size] = True
    if pages.dtype == torch.bfloat16:
        pages[~live[:, None, :].expand(pages.shape[:3])] = float("nan")
        return pages
    wide = pages.shape[3]
    d = wide // 9 * 16
    blocks = pages.view(pages.shape[0], pages.shape[1], page_size // 16, 16 * wide)
    words = blocks[..., 8 * d:].reshape(pages.shape[0], pages.shape[1], page_size, d // 16).clone()
    words[~live[:, None, :].expand(words.shape[:3])] = 0xFF      # steps and least values of 0xffff: NaN
    blocks[..., 8 * d:] = words.reshape(*blocks.shape[:3], d)
    return pages


def _cache(bits, d, hk, page, lengths, wide=None, seed=0):
    used = [-(-n // page) for n in lengths]
    wide = wide or max(max(used), 1)
    pages = sum(used) + 2
    k, v = (_store(_x(pages, hk, page, d, seed=seed + i), bits, bool(i)) for i in range(2))
    table = _table(used, wide, pages, seed)
    return _poison(k, table, lengths, page), _poison(v, table, lengths, page), table


# ---- the append ---------------------------------------------------------------------------------

def _want_append(k, v, kp, vp, table, places, cos, sin, interleaved):
    """Pages after rows [n, Hk, D] at `places` [(sequence, position)] went in; bf16, or (codes, step, least)."""
    page = kp.shape[2]
    out = []
    for x, pages, value in ((k, kp, False), (v, vp, True)):
        bf16 = pages.dtype == torch.bfloat16
        state = [pages.clone()] if bf16 else [t.clone() for t in po.unpack(pages, value)]
        for i, (b, pos) in enumerate(places):
            if pos >= table.shape[1] * page or not 0 <= int(table[b, pos // page]) < pages.shape[0]:
                continue
            row = x[i]
            if not value and cos is not None:
                row = po.turn_fp32(row, cos[pos], sin[pos], interleaved)
            new = [row] if bf16 else po.quantise(row)
            for have, want in zip(state, new):
                have[int(table[b, pos // page]), :, pos % page] = want
        out.append(state)
    return out


def _same(pages, want, value):
    got = [pages.cpu()] if pages.dtype == torch.bfloat16 else po.unpack(pages.cpu(), value)
    for x, y in zip(got, want):
        assert torch.equal(x.nan_to_num(7777.0), y.nan_to_num(7777.0))


APPENDS = [  # D, R (0: no rotation), interleaved, page, Hk, H, new tokens, lengths
    (128, 128, False, 16, 2, 16, [1, 1, 1], [0, 15, 40]),
    (64, 64, False, 64, 2, 14, [1], [63]),
    (64, 32, True, 32, 4, 4, [5, 5], [30, 0]),
    (128, 64, False, 48, 1, 3, [40, 40], [7, 48]),
    (128, 0, False, 16, 2, 2, [17, 17, 17], [0, 1, 16]),
    (64, 6, False, 16, 1, 2, [3, 3], [14, 31]),
    (128, 10, True, 16, 8, 8, [20, 20], [3, 0]),
]


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("d,r,interleaved,page,hk,h,new,lengths", APPENDS)
def test_append(cuda, bits, packed, d, r, interleaved, page, hk, h, new, lengths):
    b = len(new)
    if packed and b > 1:
        new = [new[0]] + [0] * (b - 2) + [max(1, new[0] // 2)]    # a sequence with nothing new among them
    kp, vp, table = _cache(bits, d, hk, page, [n + m for n, m in zip(new, lengths)], wide=8)
    total = sum(new)
    k, v, q = _x(total, hk, d, seed=5), _x(total, hk, d, seed=6), _x(total, h, d, seed=7)
    places = [(i, lengths[i] + j) for i in range(b) for j in range(new[i])]
    cos = sin = cos_d = sin_d = None
    if r:
        cos_d, sin_d = ktt.rotary_table(8 * page, r, device=cuda)
        cos, sin = cos_d.cpu(), sin_d.cpu()
    want = _want_append(k, v, kp, vp, table, places, cos, sin, interleaved)
    q_want = torch.stack([po.turn_fp32(q[i], cos[p], sin[p], interleaved) if r else q[i] for i, (_, p) in enumerate(places)])
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    after = torch.full_like(lens, -5)
    kd, vd, td = kp.to(cuda), vp.to(cuda), table.to(cuda)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    if packed:   # three rows behind the last sequence: neither read nor written
        ops = [torch.cat([t, torch.full((3,) + t.shape[1:], float("nan"), dtype=t.dtype)]).to(cuda) for t in (k, v, q)]
        kw = dict(cu_seq=torch.tensor(cu, dtype=torch.int32, device=cuda))
    else:
        ops = [t.view(b, new[0], t.shape[1], d).transpose(1, 2).to(cuda) for t in (k, v, q)]
        kw = {}
    out = ktt.paged_append(ops[0], ops[1], kd, vd, td, lens, cos_d, sin_d, q=ops[2], interleaved=interleaved, lengths_out=after, **kw)
    _same(kd, want[0], False)
    _same(vd, want[1], True)
    assert after.tolist() == [x + y for x, y in zip(lengths, new)] and lens.tolist() == lengths
    rows = out[:total] if packed else out.transpose(1, 2).reshape(total, h, d)
    assert torch.equal(rows.cpu(), q_want)
    if packed:   # offsets on the host: the same, without queries
        kd2, vd2 = kp.to(cuda), vp.to(cuda)
        assert ktt.paged_append(ops[0], ops[1], kd2, vd2, td, lens, cos_d, sin_d, interleaved=interleaved, cu_seq=cu) is None
        assert torch.equal(kd2.view(torch.uint8), kd.view(torch.uint8)) and torch.equal(vd2.view(torch.uint8), vd.view(torch.uint8))


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("d", [64, 128])
def test_packed_appends_of_many_sequences(cuda, bits, d):
    """Over 31 sequences, empty ones among them, with rows before the first and behind the last, against two calls of fewer."""
    hk, page, b = 2, 16, 40
    counts, lens = [(7 * i) % 4 for i in range(b)], [(5 * i) % 40 for i in range(b)]
    starts = [3]
    for n in counts:
        starts.append(starts[-1] + n)
    t = starts[-1] + 5
    k, v, q = (_x(t, h, d, seed=h + i).to(cuda) for i, h in enumerate((hk, hk, 6)))
    cos, sin = ktt.rotary_table(64, d, device=cuda)
    table = torch.randperm(b * 4, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(b, 4).to(cuda)
    lengths = torch.tensor(lens, dtype=torch.int32, device=cuda)
    cu = torch.tensor(starts, dtype=torch.int32, device=cuda)
    outs = []
    for parts in ([(0, b)], [(0, 17), (17, 31), (31, b)]):
        kp, vp = ktt.paged_cache(b * 4, hk, page, d, bits=bits, device=cuda)
        after, rows = torch.zeros(b, dtype=torch.int32, device=cuda), torch.zeros_like(q)
        for lo, hi in parts:
            got = ktt.paged_append(k, v, kp, vp, table[lo:hi], lengths[lo:hi], cos, sin, q=q, cu_seq=cu[lo:hi + 1], lengths_out=after[lo:hi])
            rows[starts[lo]:starts[hi]] = got[starts[lo]:starts[hi]]
        outs.append((kp, vp, after, rows))
    assert all(torch.equal(x, y) for x, y in zip(*outs))
    assert outs[0][2].tolist() == [x + y for x, y in zip(lens, counts)]


@pytest.mark.parametrize("bits", BITS)
def test_rows_without_a_page_go_nowhere(cuda, bits):
    """Holes in the table, a table that ends, lengths out of range: no other byte of the pool changes."""
    d, hk, page = 64, 2, 16
    kp, vp, _ = _cache(bits, d, hk, page, [64])
    table = torch.tensor([[0, -1, 2], [1, 99, 3], [-2 ** 31, 2 ** 31 - 1, -7]], dtype=torch.int32)
    k, v = _x(3, hk, 40, d, seed=1), _x(3, hk, 40, d, seed=2)
    lengths = [10, 30, -3]
    places = [(b, max(lengths[b], 0) + i) for b in range(3) for i in range(40)]
    flat = [t.transpose(1, 2).reshape(120, hk, d) for t in (k, v)]
    want = _want_append(*flat, kp, vp, table, places, None, None, False)
    kd, vd, after = kp.to(cuda), vp.to(cuda), torch.zeros(3, dtype=torch.int32, device=cuda)
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    ktt.paged_append(k.to(cuda), v.to(cuda), kd, vd, table.to(cuda), lens, lengths_out=after)
    _same(kd, want[0], False)
    _same(vd, want[1], True)
    assert after.tolist() == [48, 48, 40]    # no more than the table has room for


def test_what_four_bits_make_of_edges(cuda):
    """Groups of one value, with a NaN, with infinities, of the type's ends; rows that lie apart."""
    d, hk = 128, 1
    k = _x(8, hk, d, seed=3)
    k[0] = 0.75
    k[1, 0, 70] = float("nan")
    k[2, 0, 3] = float("inf")
    k[3] *= 1e30
    k[4] *= 1e-30
    k[5] = torch.tensor([1e-40, -1e-40]).repeat(64).to(torch.bfloat16)
    k[6, 0, :64] = -0.0
    kp, vp = ktt.paged_cache(2, hk, 16, d, bits=4, device=cuda)
    lens, table = torch.zeros(1, dtype=torch.int32, device=cuda), torch.zeros((1, 1), dtype=torch.int32, device=cuda)
    ktt.paged_append(k.to(cuda), k.to(cuda), kp, vp, table, lens, cu_seq=[0, 8])
    for pages, value in ((kp, False), (vp, True)):
        got = po.values(pages.cpu(), value)[0, 0, :8]
        want = po.worth(*po.quantise(k))[:, 0]
        assert torch.equal(torch.isfinite(got), torch.isfinite(want))
        assert torch.equal(got[torch.isfinite(want)], want[torch.isfinite(want)])
        assert torch.equal(got[0], torch.full((d,), 0.75)) and got[1, 64:].isnan().all() and torch.isfinite(got[1, :64]).all()


# ---- reading back -------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("d,hk,page,lengths", [(64, 2, 16, [0, 1, 15, 16, 17, 100]), (128, 3, 64, [200, 64]), (128, 1, 48, [47, 97])])
def test_read(cuda, bits, d, hk, page, lengths):
    kp, vp, table = _cache(bits, d, hk, page, lengths)
    cap = table.shape[1] * page
    for max_k in (None, 33):
        lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
        k, v = ktt.paged_read(kp.to(cuda), vp.to(cuda), table.to(cuda), lens, max_k=max_k)
        rows = cap if max_k is None else max_k
        assert k.shape == v.shape == (len(lengths), hk, rows, d)
        for got, pages, value in ((k, kp, False), (v, vp, True)):
            want = torch.zeros(got.shape, dtype=torch.bfloat16)
            for b, n in enumerate(lengths):
                n = min(n, rows)
                want[b, :, :n] = po.sequence(pages, table[b], n, value).to(torch.float32).to(torch.bfloat16)
            assert torch.equal(got.cpu(), want)


# ---- attention ----------------------------------------------------------------------------------

def _near(got, want, mags, sizes, dense_four_bits):
    """bf16 weights (half a step, 2^-8, of each p |v|) and a bf16 result (2^-8 of it); fp32 sums: 2^-16 of the
    terms. Over 4 bits it is p step that is rounded, before it multiplies code - 8: 2^-8 of p step |code - 8|, which can be
    more than p |v| (a value near 0 of a group far from it), so both are in `mags`. Logits: fp32 products, 2^-18 of
    sum |q| |k|. Where 4-bit keys and values become bf16 on their way (chunks
    of prompts) half a step of every key and value more: exp(2 x 2^-8 size) - 1 and 2^-8 of each p |v|."""
    e = 2.0 ** -8
    for g, w, m, z in zip(got, want, mags, sizes):
        logit = (2.0 ** -18 + (e if dense_four_bits else 0.0)) * z[..., None]
        room = e * w.abs() + (e * (2 if dense_four_bits else 1) + 2.0 ** -16 + torch.expm1(2 * logit)) * (1 + e) * m + 1e-30
        off = (g.double().cpu() - w).abs()
        assert bool((off <= room).all()), ((off - room).max().item(), off.max().item())


def _check(cuda, bits, d, h, hk, page, n, lengths, causal=True, scale=None, packed=False, seed=0, wide=None, dense_four_bits=False, **kw):
    b = len(lengths)
    counts = n if isinstance(n, list) else [n] * b
    kp, vp, table = _cache(bits, d, hk, page, lengths, seed=seed, wide=wide)
    qs = [_x(h, m, d, seed=seed + 10 + i) for i, m in enumerate(counts)]
    want, mags, sizes = po.attend([q.double() for q in qs], kp.nan_to_num(0.0) if bits == 16 else kp, vp.nan_to_num(0.0) if bits == 16 else vp,
                                  table, lengths, causal, scale or d ** -0.5)
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    args = (kp.to(cuda), vp.to(cuda), table.to(cuda), lens)
    if packed:
        cu = [0]
        for m in counts:
            cu.append(cu[-1] + m)
        out = ktt.sdpa_paged(torch.cat([q.transpose(0, 1) for q in qs]).to(cuda), *args, is_causal=causal, scale=scale, cu_seq_q=cu, **kw)
        got = [out[cu[i]:cu[i + 1]].transpose(0, 1) for i in range(b)]
    else:
        out = ktt.sdpa_paged(torch.stack(qs).to(cuda), *args, is_causal=causal, scale=scale, **kw)
        got = list(out)
    _near(got, want, mags, sizes, dense_four_bits)
    return out


TOKENS = [  # D, H, Hk, page, lengths
    (64, 14, 2, 16, [1024]),
    (64, 4, 4, 16, [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255]),
    (128, 16, 2, 16, [300, 5, 0, 129, 64]),
    (128, 32, 2, 32, [200, 77]),          # 16 rows to a key head
    (128, 6, 2, 48, [100, 250, 47]),      # pages that end inside a tile
    (64, 40, 2, 64, [130, 1]),            # more than 16 rows to a key head
    (128, 8, 8, 256, [700, 513]),
]


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("d,h,hk,page,lengths", TOKENS)
def test_single_tokens(cuda, bits, d, h, hk, page, lengths):
    _check(cuda, bits, d, h, hk, page, 1, lengths)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("n,d,h,hk,page,lengths", [
    (2, 64, 14, 2, 16, [130, 2, 1, 0]), (3, 128, 16, 4, 16, [65, 3, 64]), (8, 64, 8, 8, 32, [17, 200]), (5, 128, 32, 8, 64, [300, 4]), (9, 64, 4, 1, 16, [60, 9, 8])])
@pytest.mark.parametrize("causal", [True, False])
def test_few_tokens(cuda, bits, n, d, h, hk, page, lengths, causal):
    """Rows before a sequence's first key see nothing and are zeros."""
    _check(cuda, bits, d, h, hk, page, n, lengths, causal=causal)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("counts,d,h,hk,page,lengths", [([1, 3, 0, 7], 128, 8, 2, 16, [40, 3, 12, 100]), ([2, 1], 64, 14, 2, 32, [33, 0])])
def test_packed_queries(cuda, bits, counts, d, h, hk, page, lengths):
    _check(cuda, bits, d, h, hk, page, counts, lengths, packed=True)
    _check(cuda, bits, d, h, hk, page, counts, lengths, packed=True, max_q=max(counts), causal=False)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("packed", [False, True])
def test_chunks_of_prompts(cuda, bits, packed):
    counts = [70, 33, 130, 1] if packed else 130
    lengths = [70, 400, 130, 250] if packed else [130, 257, 100]
    _check(cuda, bits, 128, 8, 2, 32, counts, lengths, packed=packed, dense_four_bits=bits == 4)
    _check(cuda, bits, 64, 4, 4, 16, counts, lengths, packed=packed, causal=False, dense_four_bits=bits == 4, seed=3)
    _check(cuda, bits, 64, 4, 2, 64, counts, lengths, packed=packed, dense_four_bits=bits == 4, seed=5)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("d,causal", [(64, True), (128, False)])
def test_chunks_with_few_keys_or_none(cuda, bits, packed, d, causal):
    """Sequences without a key, with fewer keys than queries, and that end on a tile's last key."""
    counts = [60, 55, 1, 200, 0, 128] if packed else 60
    lengths = [0, 3, 0, 128, 40, 256] if packed else [0, 3, 60, 128]
    _check(cuda, bits, d, 6, 3, 16, counts, lengths, packed=packed, causal=causal, dense_four_bits=bits == 4)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("n", [47, 48, 49])
def test_both_sides_of_the_choice_by_tokens(cuda, bits, n):
    _check(cuda, bits, 64, 6, 2, 16, n, [60, 100], dense_four_bits=bits == 4 and n > 48)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("n", [24, 40, 64, 65])
def test_both_sides_of_the_choice_by_rows(cuda, bits, n):
    """Eight rows to a token of a K / V head, over room for many keys, and one."""
    _check(cuda, bits, 128, 16, 2, 32, n, [60, 300, 1], wide=256, dense_four_bits=bits == 4)
    _check(cuda, bits, 64, 3, 3, 32, n, [60, 300, 1], wide=256, dense_four_bits=bits == 4)


@pytest.mark.parametrize("bits", BITS)
def test_more_sequences_than_a_launch_takes(cuda, bits):
    """Over 512 sequences are several launches, dense and packed."""
    b = 700
    lengths = [i % 19 for i in range(b)]
    _check(cuda, bits, 64, 2, 1, 16, 1, lengths)
    _check(cuda, bits, 64, 2, 1, 16, [i % 2 for i in range(b)], [max(n, 1) for n in lengths], packed=True)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("d", [64, 128])
def test_more_pairs_than_ctas(cuda, bits, d):
    """One after another, whole, where no sequence is long; equal shares where one may be."""
    lengths = [(7 * i) % 50 for i in range(60)]
    _check(cuda, bits, d, 16, 16, 16, 1, lengths)
    _check(cuda, bits, d, 16, 16, 16, 1, lengths, wide=130)


@pytest.mark.parametrize("bits", BITS)
def test_one_long_sequence_among_short_ones(cuda, bits):
    _check(cuda, bits, 64, 4, 2, 16, 1, [3000, 1, 16, 40, 0, 500], seed=2)


@pytest.mark.parametrize("bits", BITS)
def test_scale_and_more_room_than_keys(cuda, bits):
    _check(cuda, bits, 64, 4, 2, 16, 1, [100, 17], scale=0.5, wide=64)
    _check(cuda, bits, 64, 4, 2, 16, 1, [100, 17], wide=64, max_k=128)
    got = [_cut(cuda, bits, n) for n in (48, None)]
    assert torch.equal(*got)


def _cut(cuda, bits, max_k):
    """max_k cuts longer sequences: the same as shorter ones."""
    kp, vp, table = _cache(bits, 64, 2, 16, [100, 17])
    lens = torch.tensor([100, 17] if max_k else [48, 17], dtype=torch.int32, device=cuda)
    return ktt.sdpa_paged(_x(2, 4, 1, 64).to(cuda), kp.to(cuda), vp.to(cuda), table.to(cuda), lens, max_k=max_k)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("d,causal", [(64, True), (64, False), (128, True), (128, False)])
def test_chunks_cut_along_their_keys(cuda, bits, packed, d, causal):
    """Few tiles and many keys: parts that end in a tile's diagonal, that no row or only some rows see, that hold one key, and
    sequences of one part or none beside them. Parts are added up in fp32: no rounding more than _near counts."""
    counts = [130, 60, 1, 0, 256, 49] if packed else 130
    _check(cuda, bits, d, 2, 1, 32, counts, [3000, 1025, 2048, 700, 2049, 49], packed=packed, causal=causal, dense_four_bits=bits == 4)
    _check(cuda, bits, d, 4, 2, 64, 1100, [1100], causal=causal, dense_four_bits=bits == 4, seed=3)
    _check(cuda, bits, d, 3, 3, 16, 50, [0, 2500], causal=causal, dense_four_bits=bits == 4, seed=4)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("d,hk", [(128, 8), (64, 16)])
def test_chunks_over_more_room_than_one_launch_takes(cuda, bits, packed, d, hk):
    """Room for 65,536 keys: the dense rows of 4 sequences are 1 GB, so 6 are two launches of 4 and 2."""
    counts = [60, 49, 0, 130, 7, 64] if packed else 60
    _check(cuda, bits, d, hk, hk, 64, counts, [100, 49, 3, 257, 0, 64], packed=packed, wide=1024, dense_four_bits=bits == 4)


@pytest.mark.parametrize("bits", BITS)
def test_pages_past_32_bits_of_a_pool(cuda, bits):
    """The same cache at the front of a small pool and at the end of one of over 4 GB."""
    d, h, hk, page, b = 128, 16, 8, 16, 2
    many = 140_000 if bits == 16 else 480_000
    small, large = (ktt.paged_cache(n, hk, page, d, bits=bits, device=cuda) for n in (8, many))
    assert large[0].numel() * large[0].element_size() > 2 ** 32
    table = torch.arange(8, dtype=torch.int32, device=cuda).view(b, 4)
    lens = torch.tensor([0, 3], dtype=torch.int32, device=cuda)
    outs = []
    for (kp, vp), t in ((small, table), (large, table + (many - 8))):
        state, out = lens, []
        for n in (50, 3, 1):
            after = torch.empty_like(state)
            ktt.paged_append(_x(b, hk, n, d, seed=n).to(cuda), _x(b, hk, n, d, seed=n + 1).to(cuda), kp, vp, t, state, lengths_out=after)
            out.append(ktt.sdpa_paged(_x(b, h, n, d, seed=n + 2).to(cuda), kp, vp, t, after))
            state = after
        outs.append(out + list(ktt.paged_read(kp, vp, t, state)))
    assert all(torch.equal(x, y) for x, y in zip(*outs)) and bool(outs[0][0].any())


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("n", [1, 4, 140])
def test_keys_without_a_page_are_zeros(cuda, bits, n):
    d, h, hk, page = 64, 4, 2, 16
    kp, vp = (_store(_x(12, hk, page, d, seed=i), bits, bool(i)) for i in range(2))
    table = torch.tensor([[3, -1, 5, 1000, 0, 2], [-1] * 6], dtype=torch.int32)
    lengths = [90, 40]
    q = _x(2, h, n, d, seed=4)
    want, mags, sizes = po.attend([x.double() for x in q], kp, vp, table, lengths, False, d ** -0.5)
    out = ktt.sdpa_paged(q.to(cuda), kp.to(cuda), vp.to(cuda), table.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda), is_causal=False)
    _near(list(out), want, mags, sizes, bits == 4 and n > 48)
    assert torch.equal(out[1], torch.zeros_like(out[1]))


@pytest.mark.parametrize("n", [1, 3, 40])
def test_pages_and_queries_in_other_orders(cuda, n):
    """bf16 pages stored [pages, page, Hk, D], keys and values in one storage, queries as head views: the same bits."""
    d, h, hk, page, lengths = 128, 8, 2, 16, [75, 40]
    kp, vp, table = _cache(16, d, hk, page, lengths)
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    q = _x(2, h, n, d, seed=4).to(cuda)
    want = ktt.sdpa_paged(q, kp.to(cuda), vp.to(cuda), table.to(cuda), lens)
    both = torch.stack([kp.transpose(1, 2), vp.transpose(1, 2)], dim=1).to(cuda)     # [pages, 2, page, Hk, D]
    k2, v2 = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    view = q.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.full((2, 9), -1, dtype=torch.int32, device=cuda)
    wide[:, :table.shape[1]] = table.to(cuda)
    got = ktt.sdpa_paged(view, k2, v2, wide[:, :table.shape[1]], lens)
    assert torch.equal(got, want)
    a, b = ktt.paged_read(k2, v2, wide, lens), ktt.paged_read(kp.to(cuda), vp.to(cuda), wide, lens)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    four = [t.to(cuda) for t in (po.pack(kp.nan_to_num(0.0), False), po.pack(vp.nan_to_num(0.0), True))]
    pool = torch.stack(four, dim=1)     # one pool for both
    assert torch.equal(ktt.sdpa_paged(q, pool[:, 0], pool[:, 1], table.to(cuda), lens), ktt.sdpa_paged(view, *four, table.to(cuda), lens))


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("b,n,cap", [(1, 1, 4096), (64, 1, 1024), (3, 2, 600), (2, 200, 500), (2, 100, 6000)])
def test_the_same_bits_every_time(cuda, bits, b, n, cap):
    """No result goes by the order in which parts of a sequence are done."""
    g = torch.Generator().manual_seed(b)
    lengths = torch.randint(cap // 2, cap + 1, (b,), generator=g).tolist()
    kp, vp, table = _cache(bits, 128, 2, 32, [1] * b, wide=-(-cap // 32))
    table = torch.randint(0, kp.shape[0], table.shape, generator=g, dtype=torch.int32)
    kp, vp = (_store(_x(kp.shape[0], 2, 32, 128, seed=i), bits, bool(i)).to(cuda) for i in range(2))
    q, lens = _x(b, 16, n, 128).to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda)
    first = ktt.sdpa_paged(q, kp, vp, table.to(cuda), lens)
    for _ in range(20):
        assert torch.equal(ktt.sdpa_paged(q, kp, vp, table.to(cuda), lens), first)
    # A neighbour changes nothing.
    lens2 = lens.clone()
    lens2[1:] = 3
    if n == 1 and b == 64:
        off = (ktt.sdpa_paged(q, kp, vp, table.to(cuda), lens2)[0].float() - first[0].float()).abs().max()
        assert off <= 2.0 ** -6 * first[0].float().abs().max()    # (cut in other places: other roundings)


# ---- together -----------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", BITS)
def test_a_model_s_run(cuda, bits):
    """Prompts of three lengths, a chunk behind them, then tokens one by one with a captured step: the cache's
    contents and every output against dense float64 attention over the keys that the cache holds."""
    d, h, hk, page, b = 64, 8, 2, 16, 3
    kp, vp = ktt.paged_cache(40, hk, page, d, bits=bits, device=cuda)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1))[:36].view(3, 12).to(device=cuda, dtype=torch.int32)
    cos, sin = ktt.rotary_table(12 * page, d, scaling="linear", factor=2.0, device=cuda)
    lens, after = torch.zeros(b, dtype=torch.int32, device=cuda), torch.zeros(b, dtype=torch.int32, device=cuda)
    have = [0] * b

    def check(out, q_rows, counts, dense):
        want, mags, sizes = po.attend([q.double() for q in q_rows], kp.cpu(), vp.cpu(), table.cpu(), have, True, d ** -0.5)
        _near(out, want, mags, sizes, dense and bits == 4)

    for step, counts in enumerate(([50, 1, 17], [40, 40, 40])):
        t = sum(counts)
        k, v, q = _x(t, hk, d, seed=step).to(cuda), _x(t, hk, d, seed=step + 20).to(cuda), _x(t, h, d, seed=step + 40).to(cuda)
        cu = [0]
        for c in counts:
            cu.append(cu[-1] + c)
        qr = ktt.paged_append(k, v, kp, vp, table, lens, cos, sin, q=q, cu_seq=cu, lengths_out=after)
        pos = torch.cat([torch.arange(have[i], have[i] + counts[i]) for i in range(b)]).to(cuda)
        q2, k2 = ktt.rotary(q, k, cos, sin, positions=pos)
        assert torch.equal(qr, q2)
        have = [x + y for x, y in zip(have, counts)]
        assert after.tolist() == have
        got_k, got_v = ktt.paged_read(kp, vp, table, after)
        for i in range(b):
            for got, rows in ((got_k, k2), (got_v, v)):
                new = rows[cu[i]:cu[i + 1]].cpu()
                new = new if bits == 16 else po.worth(*po.quantise(new)).to(torch.bfloat16)
                assert torch.equal(got[i, :, have[i] - counts[i]:have[i]].cpu(), new.transpose(0, 1))
        out = ktt.sdpa_paged(qr, kp, vp, table, after, cu_seq_q=cu)
        check([out[cu[i]:cu[i + 1]].transpose(0, 1) for i in range(b)], [qr[cu[i]:cu[i + 1]].transpose(0, 1).cpu() for i in range(b)], counts, True)
        lens.copy_(after)

    k, v, q = _x(b, hk, 1, d, seed=7).to(cuda), _x(b, hk, 1, d, seed=8).to(cuda), _x(b, h, 1, d, seed=9).to(cuda)

    def token():
        qr = ktt.paged_append(k, v, kp, vp, table, lens, cos, sin, q=q, lengths_out=after)
        out = ktt.sdpa_paged(qr, kp, vp, table, after)
        lens.copy_(after)
        return qr, out

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):   # a first call outside of the capture
        token()
    torch.cuda.current_stream().wait_stream(side)
    have = [n + 1 for n in have]
    with torch.cuda.graph(graph):
        qr, out = token()
    for step in range(3):
        for t in (k, v, q):
            t.copy_(_x(*t.shape, seed=100 + step + t.shape[1]))
        graph.replay()
        have = [n + 1 for n in have]
        assert lens.tolist() == have
        check(list(out), list(qr.cpu()), [1] * b, False)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("n", [1, 60])
def test_two_streams_and_two_graphs_at_once(cuda, bits, n):
    """Calls that run at the same time have workspaces of their own."""
    kp, vp, _ = _cache(bits, 128, 2, 32, [2000, 1500])
    table = torch.arange(2 * 40, dtype=torch.int32).view(2, 40) % kp.shape[0]
    kp, vp = (_store(_x(kp.shape[0], 2, 32, 128, seed=i), bits, bool(i)).to(cuda) for i in range(2))
    table, lens = table.to(cuda), torch.tensor([1280, 1111], dtype=torch.int32, device=cuda)
    qs = [_x(2, 16, n, 128, seed=i).to(cuda) for i in range(2)]
    want = [ktt.sdpa_paged(q, kp, vp, table, lens) for q in qs]
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(ktt.sdpa_paged(q, kp, vp, table, lens))
    torch.cuda.synchronize()
    for _ in range(10):
        eager = []
        for s, g, q in zip(streams, graphs, qs):
            with torch.cuda.stream(s):
                g.replay()
                eager.append(ktt.sdpa_paged(q, kp, vp, table, lens))
        torch.cuda.synchronize()
        for e, o, w in zip(eager, outs, want):
            assert torch.equal(e, w) and torch.equal(o, w)


@pytest.mark.parametrize("bits", BITS)
def test_first_call_of_a_kind_inside_a_capture(cuda, bits):
    """What a kernel needs set up can be set up while a stream captures: a process of its own, whose first calls are
    captured ones."""
    import subprocess
    import sys

    code = f"""
import torch, kohaku_tt_b200 as ktt
dev = torch.device("cuda:0")
kp, vp = ktt.paged_cache(8, 2, 16, 64, bits={bits}, device=dev)
table = torch.arange(8, dtype=torch.int32, device=dev).view(2, 4)
lens, after = torch.tensor([3, 40], dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
x = [torch.randn(2, h, n, 64, device=dev).bfloat16() for n in (1, 3, 50) for h in (2, 2, 8)]
cos, sin = ktt.rotary_table(64, 64, device=dev)
torch.cuda.synchronize()
def run():
    outs = []
    for i in range(3):
        q = ktt.paged_append(x[3 * i], x[3 * i + 1], kp, vp, table, lens, cos, sin, q=x[3 * i + 2], lengths_out=after)
        outs += [q, ktt.sdpa_paged(q, kp, vp, table, after), *ktt.paged_read(kp, vp, table, after), *ktt.rotary(q, x[3 * i], cos, sin)]
    return outs
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in got]
assert all(torch.equal(a, b) for a, b in zip(got, run()))
print("same")
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stdout + done.stderr[-3000:]


def test_compiled(cuda):
    kp, vp, table = _cache(16, 64, 2, 16, [20, 33], wide=4)
    kp, vp, table = kp.nan_to_num(0.0).to(cuda), vp.nan_to_num(0.0).to(cuda), table.clamp(min=0).to(cuda)
    lens, after = torch.tensor([20, 33], dtype=torch.int32, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    cos, sin = ktt.rotary_table(64, 64, device=cuda)
    k, v, q = (_x(2, x, 1, 64, seed=x).to(cuda) for x in (2, 2, 4))

    def step(q, k, v, kp, vp, after):
        q = ktt.paged_append(k, v, kp, vp, table, lens, cos, sin, q=q, lengths_out=after)
        return ktt.sdpa_paged(q, kp, vp, table, after), ktt.paged_read(kp, vp, table, after)[0]

    k2, v2, a2 = kp.clone(), vp.clone(), after.clone()
    want = step(q, k, v, kp, vp, after)
    got = torch.compile(step, fullgraph=True)(q, k, v, k2, v2, a2)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(k2, kp) and torch.equal(v2, vp) and torch.equal(a2, after)


def test_refusals(cuda):
    k, v = ktt.paged_cache(4, 2, 16, 64, device=cuda)
    table, lens = torch.zeros((2, 3), dtype=torch.int32, device=cuda), torch.ones(2, dtype=torch.int32, device=cuda)
    q, new = _x(2, 4, 1, 64).to(cuda), _x(2, 2, 1, 64).to(cuda)
    cos, sin = ktt.rotary_table(48, 64, device=cuda)
    for call in [
        lambda: ktt.sdpa_paged(q.float(), k, v, table, lens),
        lambda: ktt.sdpa_paged(q[:1], k, v, table, lens),
        lambda: ktt.sdpa_paged(q, k, v, table.long(), lens),
        lambda: ktt.sdpa_paged(q, k, v, table[:, :0], lens),
        lambda: ktt.sdpa_paged(q, k, v, table, lens.long()),
        lambda: ktt.sdpa_paged(q, k, v, table, lens[:1]),
        lambda: ktt.sdpa_paged(q, k, v[:2], table, lens),
        lambda: ktt.sdpa_paged(q[:, :, 0], k, v, table, lens),
        lambda: ktt.sdpa_paged(q[:, :, 0], k, v, table, lens, cu_seq_q=[0, 1]),
        lambda: ktt.sdpa_paged(q[:, :, 0], k, v, table, lens, cu_seq_q=[0, 2, 3]),
        lambda: ktt.sdpa_paged(q[:, :, 0], k, v, table, lens, cu_seq_q=[0, 2, 2], max_q=1),
        lambda: ktt.sdpa_paged(q, k, v, table, lens, max_k=0),
        lambda: ktt.paged_append(new, new[:, :1], k, v, table, lens),
        lambda: ktt.paged_append(new, new, k, v, table, lens, cos, None),
        lambda: ktt.paged_append(new, new, k, v, table, lens, cos[:40], sin[:40]),      # not every place of the cache
        lambda: ktt.paged_append(new, new, k, v, table, lens, cos.half(), sin.half()),
        lambda: ktt.paged_append(new, new, k, v, table, lens, q=q[:, :, :0]),
        lambda: ktt.paged_append(new, new, k, v, table, lens, lengths_out=lens),
        lambda: ktt.paged_append(new, new, k, v, table, lens, lengths_out=lens.long()),
        lambda: ktt.paged_append(new[:, :, 0], new[:, :, 0], k, v, table, lens, cu_seq=[0, 3, 2]),
    ]:
        with pytest.raises(ValueError):
            call()
    for call in [
        lambda: ktt.sdpa_paged(q, k.half(), v.half(), table, lens),
        lambda: ktt.sdpa_paged(q[:, :3], k, v, table, lens),
        lambda: ktt.sdpa_paged(q, k.view(torch.uint8)[..., :36], v.view(torch.uint8)[..., :36], table, lens),   # rows that are not dense
        lambda: ktt.sdpa_paged(q, k[:, :, :8], v[:, :, :8], table, lens),                                       # a page of 8
        lambda: ktt.sdpa_paged(q, k, v, table, lens, scale=-1.0),
        lambda: ktt.sdpa_paged(_x(2, 4, 1, 96).to(cuda), _x(4, 2, 16, 96).to(cuda), _x(4, 2, 16, 96).to(cuda), table, lens),
    ]:
        with pytest.raises(_lib.UnsupportedAttention):
            call()
    assert ktt.sdpa_paged(q[:, :, :0], k, v, table, lens).shape == (2, 4, 0, 64)
    empty = new[:, :, :0]
    after = torch.zeros_like(lens)
    ktt.paged_append(empty, empty, k, v, table, lens, lengths_out=after)
    assert after.tolist() == [1, 1]
