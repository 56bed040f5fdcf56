"""Rotary tables and rotation against float64, forward and gradient."""

import math

import pytest
import torch

import kohaku_tt_b200 as ktt
from kohaku_tt_b200.rotary import rotary_frequencies
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu


def _x(*shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _near(got, want, size):
    """A result rounded once to its type, of three fp32 operations: half a step of the value, and 4 x 2^-24 of
    the terms' magnitudes (two products, a sum, and room for the type's own subnormals)."""
    got, half = got.double().cpu(), torch.finfo(got.dtype).eps / 2
    off = (got - want).abs()
    room = half * (want.abs() + 2.0 ** -22 * size) + 2.0 ** -22 * size + torch.finfo(torch.float16).smallest_normal * 2.0 ** -11 * (half < 2.0 ** -8)
    assert bool((off <= room).all()), (off - room).max()


@pytest.mark.parametrize("positions,dim,base,how", [
    (1, 2, 10000.0, {}), (77, 64, 10000.0, {}), (4097, 100, 500000.0, dict(scaling="linear", factor=3.0)),
    (2049, 128, 10000.0, dict(scaling="base", factor=8.0)), (131072, 128, 1e6, dict(scaling="parts", factor=4.0, original=32768)),
    (300, 512, 10000.0, dict(scaling="parts", factor=1.0, original=100)),
])
def test_tables(cuda, positions, dim, base, how):
    cos, sin = ktt.rotary_table(positions, dim, base=base, device=cuda, **how)
    assert cos.shape == sin.shape == (positions, dim // 2) and cos.dtype == torch.float32
    want_c, want_s = po.table(positions, *rotary_frequencies(dim, base, **how))
    # Sines and cosines of two parts of an angle, multiplied and added: 3 ulp of values up to the scale, which is at most 2.
    for got, want in ((cos, want_c), (sin, want_s)):
        assert (got.double().cpu() - want).abs().max() <= 3 * 2.0 ** -23 * max(1.0, want.abs().max().item())


def test_frequencies_of_each_scaling():
    """The formulas, written out once more."""
    plain, one = rotary_frequencies(8, 100.0)
    assert one == 1.0 and all(math.isclose(f, 100.0 ** (-2 * i / 8)) for i, f in enumerate(plain))
    assert all(math.isclose(a, b / 5) for a, b in zip(rotary_frequencies(8, 100.0, "linear", 5.0)[0], plain))
    stretched = rotary_frequencies(8, 100.0, "base", 5.0)[0]
    assert stretched[0] == 1.0 and math.isclose(stretched[-1], plain[-1] / 5)   # the slowest pair is interpolated
    parts, scale = rotary_frequencies(128, 10000.0, "parts", 4.0, original=4096)
    whole, _ = rotary_frequencies(128, 10000.0)
    assert math.isclose(scale, 0.1 * math.log(4) + 1)
    for f, g in zip(whole, parts):
        turns = po.turns_within(f, 4096)
        assert math.isclose(g, f) if turns >= 32 else math.isclose(g, f / 4) if turns <= 1 else f / 4 < g < f


# heads, kv heads, rows, D, R, interleaved
SHAPES = [(14, 2, 77, 64, 64, False), (4, 4, 1, 128, 128, True), (3, 1, 9, 128, 64, False), (2, 2, 33, 96, 96, True), (5, 5, 7, 80, 80, False),
          (2, 1, 5, 64, 6, False), (2, 1, 5, 64, 10, True), (1, 1, 3, 50, 50, False), (1, 1, 3, 7, 6, True), (3, 2, 4, 2, 2, False), (2, 2, 3, 256, 2, True)]


@pytest.mark.parametrize("h,hk,n,d,r,interleaved", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rotation_and_gradient(cuda, h, hk, n, d, r, interleaved, dtype):
    b = 2
    q, k, dq, dk = (_x(b, x, n, d, dtype=dtype, seed=i) for i, x in enumerate((h, hk, h, hk)))
    cos, sin = ktt.rotary_table(200, r, device=cuda)
    pos = torch.randint(0, 200, (b, n), generator=torch.Generator().manual_seed(9))
    qd, kd = q.to(cuda).requires_grad_(), k.to(cuda).requires_grad_()
    yq, yk = ktt.rotary(qd, kd, cos, sin, positions=pos.to(cuda), interleaved=interleaved)
    gq, gk = torch.autograd.grad((yq, yk), (qd, kd), (dq.to(cuda), dk.to(cuda)))
    c, s = cos.cpu()[pos][:, None], sin.cpu()[pos][:, None]
    for got, x, inverse in ((yq, q, False), (yk, k, False), (gq, dq, True), (gk, dk, True)):
        assert got.dtype == dtype and got.shape == x.shape
        _near(got.detach(), *po.turn(x, c, s, interleaved, inverse))
        assert torch.equal(got.detach().cpu()[..., r:], x[..., r:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,s,d", [(1, 70, 64), (4, 4096, 128), (2, 500, 50)])
def test_products_and_sum_are_rounded_one_by_one(cuda, b, s, d, dtype, interleaved):
    """To the bit: what separate fp32 operators give. One thread's heads are four in the large call, one in the others."""
    q = _x(b, 8, s, d, dtype=dtype).to(cuda)
    cos, sin = ktt.rotary_table(s, d, device=cuda)
    x = q.float()
    x1, x2 = (x[..., ::2], x[..., 1::2]) if interleaved else (x[..., :d // 2], x[..., d // 2:])
    y1, y2 = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    want = torch.stack((y1, y2), -1).flatten(-2) if interleaved else torch.cat((y1, y2), -1)
    assert torch.equal(ktt.rotary(q, None, cos, sin, interleaved=interleaved)[0], want.to(dtype))


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_differences(cuda, interleaved):
    """fp32: the loss is linear in x, so a difference quotient is exact up to rounding: 2^-24 of the loss's terms
    over the step."""
    x, w = _x(1, 1, 4, 16, dtype=torch.float32), _x(1, 1, 4, 16, dtype=torch.float32, seed=1)
    cos, sin = ktt.rotary_table(4, 12, device=cuda)
    leaf = x.to(cuda).requires_grad_()
    (g,) = torch.autograd.grad((ktt.rotary(leaf, None, cos, sin, interleaved=interleaved)[0] * w.to(cuda)).sum(), leaf)
    for at in range(0, 64, 5):
        step = torch.zeros(64)
        step[at] = 0.5
        step = step.view_as(x)
        up, down = (ktt.rotary((x + t * step).to(cuda), None, cos, sin, interleaved=interleaved)[0].double().cpu() for t in (1, -1))
        want = ((up - down) * w.double()).sum()
        assert abs(g.flatten()[at].item() - want.item()) <= 1e-5


def test_gradient_of_the_gradient(cuda):
    """The inverse rotation's own gradient is the rotation."""
    cos, sin = ktt.rotary_table(5, 64, device=cuda)
    x = _x(1, 2, 5, 64, dtype=torch.float32).to(cuda).requires_grad_()
    w = _x(1, 2, 5, 64, dtype=torch.float32, seed=1).to(cuda).requires_grad_()
    y, _ = ktt.rotary(x, None, cos, sin)
    (g,) = torch.autograd.grad(y, x, w, create_graph=True)
    (gg,) = torch.autograd.grad(g, w, x.detach())
    assert torch.equal(gg, y.detach())


def test_one_output_used_and_one_input_wanting(cuda):
    cos, sin = ktt.rotary_table(6, 64, device=cuda)
    q, k = _x(1, 4, 6, 64).to(cuda), _x(1, 2, 6, 64, seed=1).to(cuda).requires_grad_()
    yq, yk = ktt.rotary(q, k, cos, sin)
    (gk,) = torch.autograd.grad(yk, k, yk.detach())
    want, _ = ktt.rotary(k.detach(), None, cos, -sin)
    assert torch.equal(ktt.rotary(yk.detach(), None, cos, -sin)[0], gk) and want.shape == gk.shape
    assert torch.equal(yq, ktt.rotary(q, None, cos, sin)[0])
    q2 = q.clone().requires_grad_()
    (gq,) = torch.autograd.grad(ktt.rotary(q2, k, cos, sin)[0], q2, q)
    assert torch.equal(gq, ktt.rotary(q, None, cos, -sin)[0])


def test_views_broadcasts_and_layouts(cuda):
    """A fused projection's heads, an expanded input (whose gradient is summed), packed rows, both widths of
    positions, and gradients that are expanded themselves."""
    b, n, h, d = 2, 9, 3, 64
    cos, sin = ktt.rotary_table(n, d, device=cuda)
    qkv = _x(b, n, 3 * h * d).to(cuda)
    q, k, _ = (t.view(b, n, h, d).transpose(1, 2) for t in qkv.split(h * d, -1))
    yq, yk = ktt.rotary(q, k, cos, sin)
    wq, wk = ktt.rotary(q.contiguous(), k.contiguous(), cos, sin)
    assert torch.equal(yq, wq) and torch.equal(yk, wk)
    odd = _x(b, h, n, d + 1).to(cuda)[..., 1:]     # rows that start at any 2 bytes
    assert torch.equal(ktt.rotary(odd, None, cos, sin)[0], ktt.rotary(odd.contiguous(), None, cos, sin)[0])
    turned = _x(b, d, h, n).to(cuda).permute(0, 2, 3, 1)   # columns that are no neighbours
    assert torch.equal(ktt.rotary(turned, None, cos, sin)[0], ktt.rotary(turned.contiguous(), None, cos, sin)[0])

    one = _x(b, 1, n, d, dtype=torch.float32).to(cuda).requires_grad_()
    y, _ = ktt.rotary(one.expand(b, h, n, d), None, cos, sin)
    (g,) = torch.autograd.grad(y.sum(), one)
    want, size = po.turn(torch.ones(b, 1, n, d), cos.cpu(), sin.cpu(), False, True)
    assert ((g.double().cpu() - h * want).abs() <= h * 2.0 ** -21 * size).all()

    packed = q.transpose(1, 2).reshape(b * n, h, d)
    pos = torch.arange(n, device=cuda).repeat(b)
    for p in (pos, pos.int(), pos.repeat_interleave(2)[::2]):
        yp, none = ktt.rotary(packed, None, cos, sin, positions=p)
        assert none is None and torch.equal(yp.view(b, n, h, d).transpose(1, 2), yq)
    assert torch.equal(ktt.rotary(q, k, cos, sin, positions=pos[:n])[1], yk)
    assert torch.equal(ktt.rotary(q, k, cos, sin, positions=pos[:n][None])[1], yk)


def test_columns_that_do_not_turn_are_copied(cuda):
    """NaN and infinities beside the turning columns stay where they are; positions off the table are clamped."""
    for r, interleaved in ((32, False), (32, True), (6, False), (6, True)):
        x = _x(1, 2, 3, 64)
        x[..., r:] = float("nan")
        x[..., r + 1] = float("inf")
        cos, sin = ktt.rotary_table(4, r, device=cuda)
        y, _ = ktt.rotary(x.to(cuda), None, cos, sin, interleaved=interleaved)
        assert torch.isfinite(y[..., :r]).all()
        assert torch.equal(y.cpu().view(torch.int16)[..., r:], x.view(torch.int16)[..., r:])
    x = _x(1, 1, 3, 64).to(cuda)
    cos, sin = ktt.rotary_table(4, 64, device=cuda)
    far = ktt.rotary(x, None, cos, sin, positions=torch.tensor([-7, 2, 2 ** 40], device=cuda))[0]
    assert torch.equal(far, ktt.rotary(x, None, cos, sin, positions=torch.tensor([0, 2, 3], device=cuda))[0])


def test_no_rows(cuda):
    cos, sin = ktt.rotary_table(4, 64, device=cuda)
    for shape in ((2, 3, 0, 64), (0, 3, 4, 64)):
        x = torch.empty(shape, dtype=torch.bfloat16, device=cuda)
        assert ktt.rotary(x, x, cos, sin)[1].shape == shape
    assert ktt.rotary(torch.empty((0, 3, 64), device=cuda), None, cos, sin)[0].shape == (0, 3, 64)


def test_captured_and_on_another_stream(cuda):
    cos, sin = ktt.rotary_table(64, 64, device=cuda)
    q, k = _x(2, 4, 64, 64).to(cuda), _x(2, 2, 64, 64, seed=1).to(cuda)
    want = ktt.rotary(q, k, cos, sin)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ktt.rotary(q, k, cos, sin)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other[0], want[0]) and torch.equal(other[1], want[1])
    graph = torch.cuda.CUDAGraph()
    ql = q.clone()
    with torch.cuda.graph(graph):
        got = ktt.rotary(ql, k, cos, sin)
    ql.copy_(-q)
    graph.replay()
    assert torch.equal(got[0], -want[0]) and torch.equal(got[1], want[1])


def test_compiled(cuda):
    cos, sin = ktt.rotary_table(16, 64, device=cuda)
    q, k = _x(2, 4, 16, 64).to(cuda), _x(2, 2, 16, 64, seed=1).to(cuda)
    want = ktt.rotary(q, k, cos, sin, interleaved=True)
    leaf = q.clone().requires_grad_()
    got = torch.compile(lambda a, b: ktt.rotary(a, b, cos, sin, interleaved=True), fullgraph=True)(leaf, k)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    (g,) = torch.autograd.grad(got[0], leaf, q)
    assert torch.equal(g, ktt.rotary(q, None, cos, -sin, interleaved=True)[0])
    for use in (lambda a, b: ktt.rotary(a, b, cos, sin)[1], lambda a, b: ktt.rotary(b, a, cos, sin)[0]):   # one output alone
        kl = k.clone().requires_grad_()
        (g,) = torch.autograd.grad(torch.compile(use, fullgraph=True)(q, kl), kl, k)
        assert torch.equal(g, ktt.rotary(k, None, cos, -sin)[0])


def test_the_operator_s_gradient_where_one_output_is_used(cuda):
    cos, sin = ktt.rotary_table(16, 64, device=cuda)
    q, k = _x(2, 4, 16, 64).to(cuda).requires_grad_(), _x(2, 2, 16, 64, seed=1).to(cuda).requires_grad_()
    want = ktt.rotary(k.detach(), None, cos, -sin)[0]
    out = torch.ops.ktt_b200._rotary(q, k, cos, sin, None, False, False)
    gq, gk = torch.autograd.grad(out[1], (q, k), k.detach(), allow_unused=True)
    assert torch.equal(gk, want) and (gq is None or not gq.any())


def test_refusals(cuda):
    cos, sin = ktt.rotary_table(8, 64, device=cuda)
    q, k = _x(1, 4, 8, 64).to(cuda), _x(1, 2, 8, 64).to(cuda)
    for call in [
        lambda: ktt.rotary(q, k, cos[:4], sin[:4]),                                     # tables too short
        lambda: ktt.rotary(q, k, cos.bfloat16(), sin.bfloat16()),
        lambda: ktt.rotary(q, k, cos, sin[:, :16]),
        lambda: ktt.rotary(q[..., :32], k[..., :32], cos, sin),                         # more pairs than columns
        lambda: ktt.rotary(q, k[:, :, :4], cos, sin),
        lambda: ktt.rotary(q[0, 0], None, cos, sin),
        lambda: ktt.rotary(q, k, cos, sin, positions=torch.arange(8)),                  # on the host
        lambda: ktt.rotary(q, k, cos, sin, positions=torch.arange(7, device=cuda)),
        lambda: ktt.rotary(q, k, cos, sin, positions=torch.arange(8., device=cuda)),
        lambda: ktt.rotary(q, k, cos.clone().requires_grad_(), sin),
        lambda: ktt.rotary_table(0, 64), lambda: ktt.rotary_table(4, 63), lambda: ktt.rotary_table(4, 514),
        lambda: ktt.rotary_table(4, 64, scaling="parts", factor=2.0), lambda: ktt.rotary_table(4, 64, scaling="other"),
        lambda: ktt.rotary_table(4, 64, factor=-1.0, scaling="linear"),
    ]:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        ktt.rotary(q.double(), k.double(), cos, sin)
    with pytest.raises(NotImplementedError):
        ktt.rotary(q, k.float(), cos, sin)
    with pytest.raises(RuntimeError):
        ktt.rotary(q.cpu(), None, cos.cpu(), sin.cpu())
