"""Rotation by positions of several axes, forward and gradient, alone and in the append, against float64."""

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


def _x(*shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _near(got, want, size):
    """A result rounded once to its type, of three fp32 operations: half a step of the value, and 4 x 2^-24 of
    the terms' magnitudes (two products, a sum, and room for the type's own subnormals)."""
    got, half = got.double().cpu(), torch.finfo(got.dtype).eps / 2
    off = (got - want).abs()
    room = half * (want.abs() + 2.0 ** -22 * size) + 2.0 ** -22 * size + torch.finfo(torch.float16).smallest_normal * 2.0 ** -11 * (half < 2.0 ** -8)
    assert bool((off <= room).all()), (off - room).max()


def _axes(kind, pairs, axes):
    g = torch.Generator().manual_seed(pairs)
    if kind == "runs":
        return tuple(min(axes - 1, i * axes // pairs) for i in range(pairs))
    if kind == "turns":
        return tuple(i % axes for i in range(pairs))
    return tuple(torch.randint(0, axes, (pairs,), generator=g).tolist())


# heads, kv heads, rows, D, R, interleaved
SHAPES = [(14, 2, 77, 64, 64, False), (4, 4, 1, 128, 128, True), (3, 1, 9, 128, 64, False), (2, 2, 33, 96, 96, True), (5, 5, 7, 80, 80, False),
          (2, 1, 5, 64, 6, False), (2, 1, 5, 64, 10, True), (1, 1, 3, 7, 6, True), (3, 2, 4, 2, 2, False), (1, 1, 2, 1024, 1024, False)]


@pytest.mark.parametrize("h,hk,n,d,r,interleaved", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kind,axes", [("runs", 3), ("turns", 3), ("any", 4), ("any", 2), ("runs", 1)])
def test_rotation_and_gradient(cuda, path, h, hk, n, d, r, interleaved, dtype, kind, axes):
    b = 2
    q, k, dq, dk = (_x(b, x, n, d, dtype=dtype, seed=i) for i, x in enumerate((h, hk, h, hk)))
    cos, sin = ktt.rotary_table(200, min(r, 512), device=cuda)
    if r > 512:
        cos, sin = (torch.cat([t, t.flip(0)], 1) for t in (cos, sin))
    of_pair = _axes(kind, r // 2, axes)
    pos = torch.randint(-3, 203, (axes, b, n), generator=torch.Generator().manual_seed(9))     # (clamped to the tables)
    qd, kd = q.to(cuda).requires_grad_(), k.to(cuda).requires_grad_()
    yq, yk = ktt.rotary(qd, kd, cos, sin, positions=pos.to(cuda), interleaved=interleaved, axes=of_pair)
    gq, gk = torch.autograd.grad((yq, yk), (qd, kd), (dq.to(cuda), dk.to(cuda)))
    c, s = (t[:, None] for t in so.axis_rows(cos.cpu(), sin.cpu(), pos, of_pair))
    for got, x, inverse in ((yq, q, False), (yk, k, False), (gq, dq, True), (gk, dk, True)):
        assert got.dtype == dtype and got.shape == x.shape
        _near(got.detach(), *po.turn(x, c, s, interleaved, inverse))
        assert torch.equal(got.detach().cpu()[..., r:], x[..., r:])
    assert torch.equal(yq.detach().cpu(), po.turn_fp32(q, c, s, interleaved))      # to the bit


@pytest.mark.parametrize("interleaved", [False, True])
def test_many_rows(cuda, interleaved):
    """As many threads as have four heads each; packed, positions of 64 bits and of any strides, queries and keys in one storage."""
    t, h, hk, d = 5000, 12, 4, 128
    both = _x(t, h + hk, d, seed=1)
    of_pair, pos = _axes("turns", 32, 3), torch.randint(0, 300, (t, 3), generator=torch.Generator().manual_seed(2))
    cos, sin = ktt.rotary_table(300, 64, device=cuda)
    x = both.to(cuda)
    yq, yk = ktt.rotary(x[:, :h], x[:, h:], cos, sin, positions=pos.to(cuda).t(), interleaved=interleaved, axes=of_pair)
    c, s = (y[:, None] for y in so.axis_rows(cos.cpu(), sin.cpu(), pos.t(), of_pair))
    assert torch.equal(torch.cat([yq, yk], 1).cpu(), po.turn_fp32(both, c, s, interleaved))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,h,hk,d,r,dtype", [(5200, 13, 3, 128, 128, torch.bfloat16), (70000, 9, 5, 64, 64, torch.float16), (80000, 18, 3, 128, 96, torch.bfloat16),
                                              (40000, 5, 1, 80, 80, torch.float32), (30000, 33, 1, 72, 64, torch.bfloat16), (20000, 10, 10, 64, 20, torch.bfloat16)])
def test_threads_with_many_heads_are_threads_with_one(cuda, interleaved, t, h, hk, d, r, dtype):
    """Rows in one call, whose threads go through several groups of heads, against the same rows a few at a time; one axis and three."""
    g = torch.Generator(device=cuda).manual_seed(1)
    q, k = torch.randn((t, h, d), generator=g, device=cuda).to(dtype), torch.randn((t, hk, d), generator=g, device=cuda).to(dtype)
    cos, sin = ktt.rotary_table(500, r, device=cuda)
    pos, some = torch.randint(0, 500, (3, t), generator=g, device=cuda), torch.tensor([0, 1, t // 2, t - 2, t - 1], device=cuda)
    for at, axes in ((pos[0], None), (pos, _axes("turns", r // 2, 3))):
        got = ktt.rotary(q, k, cos, sin, positions=at, interleaved=interleaved, axes=axes)
        want = ktt.rotary(q[some], k[some], cos, sin, positions=at[..., some], interleaved=interleaved, axes=axes)
        assert torch.equal(got[0][some], want[0]) and torch.equal(got[1][some], want[1])
        c, s = (cos[at], sin[at]) if axes is None else so.axis_rows(cos, sin, at, axes)
        whole = [po.turn_fp32(x, c[:, None], s[:, None], interleaved) for x in (q, k)]
        assert torch.equal(got[0], whole[0]) and torch.equal(got[1], whole[1])


def test_alike_positions_are_those_of_one_axis(cuda, path):
    """Text: all axes count on together. [axes, S] and [axes, 1, S] serve all batch entries."""
    q, k = _x(3, 8, 40, 64, seed=1).to(cuda), _x(3, 2, 40, 64, seed=2).to(cuda)
    cos, sin = ktt.rotary_table(64, 64, device=cuda)
    at = torch.arange(7, 47, dtype=torch.int32, device=cuda)
    want = ktt.rotary(q, k, cos, sin, positions=at)
    for pos in (at.expand(3, 40), at.expand(3, 1, 40), at.expand(3, 3, 40), at.expand(4, 40).long()):
        got = ktt.rotary(q, k, cos, sin, positions=pos, axes=[i % 3 for i in range(32)])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_gradient_by_differences_and_of_the_gradient(cuda, path):
    """The rotation is linear: differences are exact up to rounding, and the gradient's gradient is the rotation."""
    q = _x(1, 2, 6, 16, dtype=torch.float32, seed=3).to(cuda).requires_grad_()
    cos, sin = ktt.rotary_table(32, 12, device=cuda)
    pos, of_pair = torch.randint(0, 32, (3, 6), generator=torch.Generator().manual_seed(4)).to(cuda), (0, 1, 2, 2, 1, 0)
    w = _x(1, 2, 6, 16, dtype=torch.float32, seed=5).to(cuda)

    def f(x):
        return ktt.rotary(x, None, cos, sin, positions=pos, axes=of_pair)[0]

    (g,) = torch.autograd.grad(f(q), q, w, create_graph=True)
    step = _x(1, 2, 6, 16, dtype=torch.float32, seed=6).to(cuda)
    with torch.no_grad():
        change = ((f(q + step) - f(q - step)).double() * w.double()).sum() / 2
        # (192 terms, each off by some 2^-22 of products of about 1)
        assert abs(change - (g.double() * step.double()).sum()) <= 192 * 2.0 ** -20
    v = w.clone().requires_grad_()
    (g2,) = torch.autograd.grad(f(q), q, v, create_graph=True)
    (back,) = torch.autograd.grad(g2, v, step)
    assert torch.equal(back, f(step))
    (only,) = torch.autograd.grad(ktt.rotary(q, q.detach(), cos, sin, positions=pos, axes=of_pair)[0].sum(), q)
    assert torch.equal(only, torch.autograd.grad(f(q).sum(), q)[0])


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d,pairs,interleaved", [(128, 64, False), (64, 16, True), (64, 5, False)])
@pytest.mark.parametrize("packed", [False, True])
def test_append(cuda, path, bits, d, pairs, interleaved, packed):
    """Rows turned by their own positions, one axis and three, are those that `rotary` makes, at their places."""
    b, n, h, hk, page = 3, 19, 6, 2, 16
    lengths = torch.tensor([0, 15, 33], dtype=torch.int32, device=cuda)
    k, v, q = _x(b * n, hk, d, seed=1).to(cuda), _x(b * n, hk, d, seed=2).to(cuda), _x(b * n, h, d, seed=3).to(cuda)
    cos, sin = ktt.rotary_table(20, 2 * pairs, device=cuda)      # (fewer rows than places)
    table = torch.randperm(24, generator=torch.Generator().manual_seed(4)).view(3, 8)[:, :4].to(device=cuda, dtype=torch.int32).contiguous()
    three = torch.randint(0, 20, (3, b * n), generator=torch.Generator().manual_seed(5)).to(cuda)
    for pos, axes in ((three[0].int(), None), (three, _axes("any", pairs, 3))):
        want_q, want_k = ktt.rotary(q, k, cos, sin, positions=pos, interleaved=interleaved, axes=axes)
        plain = ktt.paged_cache(24, hk, page, d, bits=bits, device=cuda)
        got = ktt.paged_cache(24, hk, page, d, bits=bits, device=cuda)
        cu = torch.arange(0, b * n + 1, n, dtype=torch.int32, device=cuda)
        ktt.paged_append(want_k, v, *plain, table, lengths, cu_seq=cu)
        if packed:
            out = ktt.paged_append(k, v, *got, table, lengths, cos, sin, q=q, interleaved=interleaved, cu_seq=cu, positions=pos, axes=axes)
        else:
            rows = [x.view(b, n, -1, d).transpose(1, 2) for x in (k, v, q)]
            out = ktt.paged_append(rows[0], rows[1], *got, table, lengths, cos, sin, q=rows[2], interleaved=interleaved, axes=axes,
                                   positions=pos.view(*pos.shape[:-1], b, n))
            out = out.transpose(1, 2).reshape(b * n, h, d)
        assert torch.equal(out, want_q)
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(plain, got))


@pytest.mark.parametrize("bits,d,h,hk,r,batch,tokens", [(16, 128, 13, 4, 128, 3, 1500), (4, 128, 12, 4, 64, 40, 4100), (16, 64, 14, 2, 64, 5, 12000), (4, 128, 33, 3, 128, 2, 7000),
                                                        (4, 64, 9, 9, 32, 33, 21000), (16, 128, 16, 2, 20, 2, 6000)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_of_many_rows(cuda, bits, d, h, hk, r, batch, tokens, interleaved):
    """Threads with several groups of heads, and queries by pairs: rows are those that `rotary` makes, at their places; packed rows of no sequence
    are left, those of few sequences and of many are found."""
    g = torch.Generator(device=cuda).manual_seed(1)
    k, v, q = (torch.randn((tokens, x, d), generator=g, device=cuda).to(torch.bfloat16) for x in (hk, hk, h))
    cut = torch.randint(0, tokens - 7, (batch - 1,), generator=torch.Generator().manual_seed(2)).sort().values.tolist()
    cu = torch.tensor([0, *cut, tokens - 7], dtype=torch.int32, device=cuda)
    counts = (cu[1:] - cu[:-1]).tolist()
    lengths, page = torch.randint(0, 40, (batch,), generator=torch.Generator().manual_seed(3)).to(device=cuda, dtype=torch.int32), 16
    wide = max(-(-(n + 40) // page) for n in counts)
    used = [-(-(n + int(m)) // page) for n, m in zip(counts, lengths)]
    table, names = torch.full((batch, wide), -1, dtype=torch.int32), torch.randperm(sum(used), generator=torch.Generator().manual_seed(4)).to(torch.int32)
    for i, n in enumerate(used):
        table[i, :n] = names[sum(used[:i]):sum(used[:i]) + n]
    table = table.to(cuda)
    cos, sin = ktt.rotary_table(wide * page, r, device=cuda)
    at = torch.cat([torch.arange(n) + int(m) for n, m in zip(counts, lengths)] + [torch.zeros(7, dtype=torch.int64)]).to(cuda)
    three = torch.randint(0, wide * page, (3, tokens), generator=g, device=cuda)
    for pos, axes in ((None, None), (three, _axes("turns", r // 2, 3))):
        want_q, want_k = ktt.rotary(q, k, cos, sin, positions=at if pos is None else pos, interleaved=interleaved, axes=axes)
        plain, got = (ktt.paged_cache(sum(used), hk, page, d, bits=bits, device=cuda) for _ in range(2))
        bounds = ktt.paged_bounds(got[0], table, lengths)
        for b in range(batch):      # a sequence at a time, in lots of few rows
            for i in range(0, counts[b], 300):
                rows = slice(int(cu[b]) + i, int(cu[b]) + min(i + 300, counts[b]))
                ktt.paged_append(want_k[rows].transpose(0, 1)[None], v[rows].transpose(0, 1)[None], *plain, table[b:b + 1], lengths[b:b + 1] + i)
        out = ktt.paged_append(k, v, *got, table, lengths, cos, sin, q=q, interleaved=interleaved, cu_seq=cu, positions=pos, axes=axes, bounds=bounds)
        assert torch.equal(out[:-7], want_q[:-7])
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(plain, got))
        after = lengths + (cu[1:] - cu[:-1])
        assert torch.equal(bounds, ktt.paged_bounds(plain[0], table, after))


def test_compiled(cuda):
    """One graph, queries and keys, both gradients and one alone."""
    cos, sin = ktt.rotary_table(16, 64, device=cuda)
    q, k = _x(2, 4, 16, 64).to(cuda), _x(2, 2, 16, 64, seed=1).to(cuda)
    at, axes = torch.randint(0, 16, (3, 2, 16), generator=torch.Generator().manual_seed(2)).to(cuda), _axes("turns", 32, 3)

    def turned(a, b):
        return ktt.rotary(a, b, cos, sin, positions=at, axes=axes)

    ql, kl = q.clone().requires_grad_(), k.clone().requires_grad_()
    want = turned(ql, kl)
    got = torch.compile(turned, fullgraph=True)(ql, kl)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    a, b = torch.autograd.grad(want, (ql, kl), (q, k), retain_graph=True), torch.autograd.grad(got, (ql, kl), (q, k))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    (a,), (b,) = torch.autograd.grad(want[1], kl, k), torch.autograd.grad(torch.compile(lambda x: turned(q, x)[1], fullgraph=True)(kl), kl, k)
    assert torch.equal(a, b)
    # An append by such positions, without bounds.
    table, lens = torch.arange(4, dtype=torch.int32, device=cuda).view(2, 2), torch.zeros(2, dtype=torch.int32, device=cuda)
    pages, same = ktt.paged_cache(4, 2, 16, 64, device=cuda), ktt.paged_cache(4, 2, 16, 64, device=cuda)

    def append(kp, vp):
        return ktt.paged_append(k, k, kp, vp, table, lens, cos, sin, q=q, positions=at, axes=axes)

    assert torch.equal(torch.compile(append, fullgraph=True)(*pages), append(*same)) and torch.equal(pages[0], same[0])
    out = torch.ops.ktt_b200._rotary_axes(ql, kl, cos, sin, at, False, False, list(axes))
    assert torch.equal(torch.autograd.grad(out[1], kl, k)[0], a)


def test_refusals(cuda, path):
    q = _x(2, 2, 5, 8).to(cuda)
    cos, sin = ktt.rotary_table(9, 8, device=cuda)
    at = torch.zeros((3, 5), dtype=torch.int32, device=cuda)
    for kw in (dict(axes=(0, 1, 2, 0)), dict(axes=(0, 1, 2), positions=at), dict(axes=(0, 1, 3, 0), positions=at), dict(axes=(0, -1, 0, 0), positions=at),
               dict(axes=(0, 1, 2, 0), positions=at.float()), dict(axes=(0, 1, 2, 0), positions=at[:, :4]), dict(axes=(0, 1, 2, 0), positions=at[0]),
               dict(positions=at), dict(axes=(0, 0, 0, 0), positions=torch.zeros((5, 5), dtype=torch.int32, device=cuda))):
        with pytest.raises(ValueError):
            ktt.rotary(q, None, cos, sin, **kw)
    pages, table, n = ktt.paged_cache(4, 2, 16, 64, device=cuda), torch.zeros((2, 2), dtype=torch.int32, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    k, (cos, sin) = _x(2, 2, 5, 64).to(cuda), ktt.rotary_table(32, 8, device=cuda)
    for kw in (dict(positions=at[0]), dict(cos=cos, sin=sin, axes=(0, 1, 2, 0)), dict(cos=cos, sin=sin, positions=at[0], axes=(0, 0, 0)),
               dict(cos=cos, sin=sin, positions=at[0, :3]), dict(bounds=torch.zeros((4, 2, 2, 64), device=cuda)),
               dict(bounds=torch.zeros((4, 2, 2, 128), dtype=torch.bfloat16, device=cuda))):
        with pytest.raises(ValueError):
            ktt.paged_append(k, k, *pages, table, n, **kw)
