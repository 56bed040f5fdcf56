"""The serving operators together: tables, append by positions of several axes with bounds, selection and attention, step by
step; captured and replayed, on other streams, compiled."""

import pytest
import torch

import kohaku_tt_b200 as ktt
from oracle import serving_oracle as so

pytestmark = pytest.mark.gpu


def _x(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def _i32(x, cuda):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


class Server:
    """A cache of `batch` sequences with everything that a step reads and writes."""

    def __init__(self, cuda, batch=3, bits=16, d=64, h=8, hk=2, page=16, wide=20, pool=50):
        self.page, self.h, self.hk, self.d = page, h, hk, d
        self.kp, self.vp = ktt.paged_cache(pool, hk, page, d, bits=bits, device=cuda)
        self.table = torch.full((batch, wide), -1, dtype=torch.int32, device=cuda)
        self.free = torch.randperm(pool, generator=torch.Generator().manual_seed(1)).to(device=cuda, dtype=torch.int32)
        self.count, self.left = _i32([pool], cuda), _i32([0], cuda)
        self.lengths, self.after = _i32([0] * batch, cuda), _i32([0] * batch, cuda)
        self.bounds = ktt.paged_bounds(self.kp, self.table, self.lengths)
        self.cos, self.sin = ktt.rotary_table(wide * page, d, device=cuda)
        self.axes = tuple(i % 3 for i in range(d // 2))

    def step(self, q, k, v, added, positions, top=5):
        cu, at, slots, granted = ktt.paged_reserve(self.table, self.lengths, added, self.free, self.count, self.page, q.shape[0], self.left)
        q = ktt.paged_append(k, v, self.kp, self.vp, self.table, self.lengths, self.cos, self.sin, q=q, cu_seq=cu, lengths_out=self.after,
                             positions=positions + at, axes=self.axes, bounds=self.bounds)
        chosen, keys = ktt.paged_select(q, self.bounds, self.table, self.after, self.page, top, first=1, last=2, cu_seq_q=cu)
        out = ktt.sdpa_paged(q, self.kp, self.vp, chosen, keys)
        self.lengths.copy_(self.after)
        self.count.copy_(self.left)
        return q, chosen, keys, out, slots, granted


def _near(got, want, mag, size):
    """As in the tests of attention over tables of a token's own."""
    e = 2.0 ** -8
    room = e * want.abs() + (e + 2.0 ** -16 + torch.expm1(2 * 2.0 ** -18 * size[..., None])) * (1 + e) * mag + 1e-30
    off = (got.double().cpu() - want).abs()
    assert bool((off <= room).all()), (off - room).max().item()


def _rows(t, s, seed):
    return _x(t, s.h, s.d, seed=seed), _x(t, s.hk, s.d, seed=seed + 1), _x(t, s.hk, s.d, seed=seed + 2)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d", [64, 128])
def test_prompts_then_tokens(cuda, bits, d):
    s = Server(cuda, bits=bits, d=d)
    have = [0, 0, 0]
    for i, added in enumerate(([150, 3, 40], [1, 1, 1], [1, 60, 1], [1, 1, 1], [4, 1, 0])):
        t = sum(added)
        q, k, v = _rows(t, s, 10 * i)
        shift = torch.randint(0, 3, (3, t), generator=torch.Generator().manual_seed(i)).to(torch.int32)
        turned, chosen, keys, out, slots, granted = s.step(q.to(cuda), k.to(cuda), v.to(cuda), _i32(added, cuda), shift.to(cuda))
        at = torch.tensor([n + j for n, m in zip(have, added) for j in range(m)])
        want_q, want_k = ktt.rotary(q.to(cuda), k.to(cuda), s.cos, s.sin, positions=(at + shift).to(cuda), axes=s.axes)
        assert torch.equal(turned, want_q) and granted.tolist() == added
        if bits == 16:      # the slots are where the rows lie
            assert torch.equal(s.kp.transpose(1, 2).flatten(0, 1)[slots], want_k)
        have = [x + y for x, y in zip(have, added)]
        assert s.lengths.tolist() == have and s.count.item() == 50 - sum(-(-n // 16) for n in have)
        table, bounds = s.table.cpu(), so.bounds(s.kp.cpu(), s.table.cpu(), have, torch.zeros_like(s.bounds).cpu())
        assert torch.equal(s.bounds.cpu(), bounds)
        owners = so.tokens(added, have, 320)
        want, want_keys = so.select(turned.cpu(), bounds, table, owners, 16, 5, 1, 2)
        assert torch.equal(chosen.cpu(), want) and torch.equal(keys.cpu(), want_keys)
        some = [0, t // 2, t - 1]
        _near(out[some], *so.attend(turned.cpu()[some], s.kp.cpu(), s.vp.cpu(), want[some], want_keys[some], d ** -0.5))


@pytest.mark.parametrize("bits", [16, 4])
def test_captured_steps_are_eager_steps(cuda, bits):
    """One token of each sequence, captured once and replayed, against the same steps one by one."""
    a, b = Server(cuda, bits=bits), Server(cuda, bits=bits)
    q, k, v = (x.to(cuda) for x in _rows(90, a, 1))
    added = _i32([60, 10, 20], cuda)
    shift = torch.zeros((3, 90), dtype=torch.int32, device=cuda)
    for s in (a, b):
        s.step(q, k, v, added, shift)
    one, rows, shift = _i32([1, 1, 1], cuda), [torch.zeros_like(x[:3]) for x in (q, k, v)], shift[:, :3].contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):      # (kernels are set up; then the state again as it was)
        kept = [x.clone() for x in (a.kp, a.vp, a.table, a.count, a.lengths, a.bounds)]
        a.step(*rows, one, shift)
        for x, y in zip((a.kp, a.vp, a.table, a.count, a.lengths, a.bounds), kept):
            x.copy_(y)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = a.step(*rows, one, shift)
    for i in range(20):
        new = [x.to(cuda) for x in _rows(3, a, 100 + 3 * i)]
        for x, y in zip(rows, new):
            x.copy_(y)
        graph.replay()
        want = b.step(*new, one, shift)
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        assert torch.equal(a.bounds, b.bounds) and torch.equal(a.table, b.table) and a.count.item() == b.count.item()


@pytest.mark.parametrize("bits", [16, 4])
def test_pools_past_32_bits(cuda, bits):
    """Pages and bounds that lie more than 2^32 bytes (bounds: 2^31 values) behind the first: as in a small pool."""
    d, h, hk, page, wide, pool = 128, 16, 8, 64, 6, 20000
    row = d if bits == 16 else d // 2 + d // 16
    kind = torch.bfloat16 if bits == 16 else torch.uint8
    small = [torch.zeros((2 * wide, hk, page, row), dtype=kind, device=cuda) for _ in range(2)]
    stride = 2 ** 18 if bits == 16 else 2 ** 18 + 16      # of a page, in bytes
    big = torch.empty(pool * stride + 2 ** 18, dtype=torch.uint8, device=cuda).view(kind)
    per = stride // big.element_size()
    large = [big.as_strided((pool, hk, page, row), (per, page * row, row, 1), i * hk * page * row) for i in range(2)]
    names = torch.tensor([[19999, 0, 16390, 8200, 19000, 3], [17000, 18000, 19990, 1, 16400, 12000]], dtype=torch.int32, device=cuda)
    table = torch.arange(2 * wide, dtype=torch.int32, device=cuda).view(2, wide)
    wider = torch.empty(pool * 2 ** 17, dtype=torch.bfloat16, device=cuda)
    far = wider.as_strided((pool, hk, 2, d), (2 ** 17, 2 * d, d, 1))
    near = torch.zeros((2 * wide, hk, 2, d), dtype=torch.bfloat16, device=cuda)
    cos, sin = ktt.rotary_table(wide * page, d, device=cuda)
    have, after = _i32([0, 0], cuda), _i32([0, 0], cuda)
    for i, added in enumerate(([300, 77], [1, 1], [5, 200])):
        t = sum(added)
        q, k, v = (x.to(cuda) for x in (_x(t, h, d, seed=i), _x(t, hk, d, seed=i + 9), _x(t, hk, d, seed=i + 18)))
        cu = _i32([0, added[0], t], cuda)
        results = []
        for (kp, vp), names_of, bounds in ((small, table, near), (large, names, far)):
            turned = ktt.paged_append(k, v, kp, vp, names_of, have, cos, sin, q=q, cu_seq=cu, lengths_out=after, bounds=bounds)
            chosen, keys = ktt.paged_select(turned, bounds, names_of, after, page, 3, cu_seq_q=cu)
            results.append((turned, chosen, keys, ktt.sdpa_paged(turned, kp, vp, chosen, keys)))
        (turned, chosen, keys, out), (other, chosen_far, keys_far, out_far) = results
        assert torch.equal(turned, other) and torch.equal(keys, keys_far) and torch.equal(out, out_far)
        assert torch.equal(torch.where(chosen >= 0, names.flatten()[chosen.clamp(min=0).long()], -1), chosen_far)
        have.copy_(after)
    assert torch.equal(near[table.long()][:, :5], far[names.long()][:, :5])
    assert torch.equal(ktt.paged_bounds(large[0], names, have, bounds=torch.empty_like(wider).as_strided(far.shape, far.stride()))[names.long()][:, :5], near[table.long()][:, :5])


def test_two_streams_and_two_graphs_at_once(cuda):
    """Calls share nothing: what runs beside another is as it is alone."""
    d, h, hk, page, wide, top = 128, 16, 2, 16, 400, 40
    data = []
    for i in range(2):
        x = _x(2 * wide, hk, page, d, seed=i).to(cuda)
        table = torch.randperm(2 * wide, generator=torch.Generator().manual_seed(i)).view(2, wide).to(device=cuda, dtype=torch.int32)
        data.append((_x(2, h, 1, d, seed=5 + i).to(cuda), x, table, _i32([wide * page, wide * page - 77 * i], cuda)))

    def run(q, pages, table, lens):
        bounds = ktt.paged_bounds(pages, table, lens)
        chosen, keys = ktt.paged_select(q, bounds, table, lens, page, top)
        return chosen, ktt.sdpa_paged(q, pages, pages, chosen, keys)

    want = [run(*x) for x in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, got = [], []
    for x in data:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(run(*x))
    for _ in range(20):
        outs = []
        for s, g, x in zip(streams, graphs, data):
            with torch.cuda.stream(s):
                g.replay()
        for s, x in zip(reversed(streams), data):
            with torch.cuda.stream(s):
                outs.append(run(*x))
        torch.cuda.synchronize()
        for a, b, c in zip(got, outs, want):
            assert all(torch.equal(x, z) and torch.equal(y, z) for x, y, z in zip(a, b, c))


def test_compiled_whole(cuda):
    """The step in one graph of torch.compile, against the eager one; and a rotation's gradient."""
    a, b = Server(cuda), Server(cuda)
    q, k, v = (x.to(cuda) for x in _rows(40, a, 1))
    added, shift = _i32([30, 10, 0], cuda), torch.zeros((3, 40), dtype=torch.int32, device=cuda)
    want = a.step(q, k, v, added, shift)
    kept, kept_left = torch.tensor([30, 4, 0], dtype=torch.int32, device=cuda), _i32([0], cuda)
    ktt.paged_release(a.table, a.lengths, kept, a.free, a.count, 16, kept_left)

    def step(s, q, k, v, added, shift):
        cu, at, slots, granted = ktt.paged_reserve(s.table, s.lengths, added, s.free, s.count, s.page, 40, s.left)
        q = ktt.paged_append(k, v, s.kp, s.vp, s.table, s.lengths, s.cos, s.sin, q=q, cu_seq=cu, lengths_out=s.after, positions=shift + at, axes=s.axes, bounds=s.bounds)
        chosen, keys = ktt.paged_select(q, s.bounds, s.table, s.after, s.page, 5, first=1, last=2, cu_seq_q=cu)
        again = ktt.paged_bounds(s.kp, s.table, s.after, bounds=torch.zeros_like(s.bounds))
        out = ktt.sdpa_paged(q, s.kp, s.vp, chosen, keys)
        left = torch.zeros_like(s.count)
        ktt.paged_release(s.table, s.after, kept, s.free, s.left, s.page, left)
        return q, chosen, keys, out, slots, granted, again, left

    got = torch.compile(step, fullgraph=True)(b, q, k, v, added, shift)
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    assert torch.equal(got[6], b.bounds) and torch.equal(a.bounds, b.bounds) and torch.equal(a.table, b.table) and got[7].item() == kept_left.item()

    x = _x(2, 4, 9, 64, seed=7).to(cuda).requires_grad_()
    at = torch.randint(0, 99, (3, 9), generator=torch.Generator().manual_seed(8)).to(cuda)

    def turned(x):
        return ktt.rotary(x, None, a.cos, a.sin, positions=at, axes=a.axes)[0].square().sum()

    (want,) = torch.autograd.grad(turned(x), x)
    (got,) = torch.autograd.grad(torch.compile(turned, fullgraph=True)(x), x)
    assert torch.equal(got, want)


def test_the_gradient_captured_beside_an_eager_graph(cuda):
    """A captured forward and backward of a rotation by axes, while an eager graph of other leaves lives."""
    s = Server(cuda)
    x = _x(1, 4, 9, 64, seed=7).to(cuda).requires_grad_()
    other = _x(1, 4, 9, 64, seed=8).to(cuda).requires_grad_()
    at, w = torch.arange(27, device=cuda).view(3, 9), _x(1, 4, 9, 64, seed=9).to(cuda)
    alive = ktt.rotary(other, None, s.cos, s.sin, positions=at, axes=s.axes)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ktt.rotary(x, None, s.cos, s.sin, positions=at, axes=s.axes)[0]
        (want,) = torch.autograd.grad(y, x, w)
    torch.cuda.current_stream().wait_stream(side)
    del y
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(ktt.rotary(x, None, s.cos, s.sin, positions=at, axes=s.axes)[0], x, w)
    graph.replay()
    assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(alive, other, w)[0], want)
