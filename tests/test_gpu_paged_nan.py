"""Attention over pages where a query or a key is no number: it shows in the rows that it reaches and in no other, whichever
way a call takes."""

import pytest
import torch

import kohaku_tt_b200 as ktt
from kohaku_tt_b200 import ops
from oracle import paged_oracle as po
from tests.launched import launched
from tests.test_gpu_paged import _poison, _store, _table, _x

pytestmark = pytest.mark.gpu

BITS = [16, 4]
NAN, INF = float("nan"), float("inf")
# D, H, Hk, tokens, lengths, whether the keys of the call's tiles are cut into parts (None: not a matter of tiles)
CASES = [
    (128, 2, 1, 130, [3000, 1025], True),
    (64, 2, 1, 130, [3000, 1025], True),
    (128, 8, 2, 130, [300, 257], False),
    (64, 8, 2, 130, [300, 257], False),
    (128, 16, 2, 4, [3000, 1025], None),
    (64, 14, 2, 1, [9000, 40], None),
    (128, 16, 2, 1, [9000, 40], None),
]


class _Run:
    """One cache and one call over it, dense or packed."""

    def __init__(self, cuda, bits, d, h, hk, n, lengths, packed, causal=True):
        page = 32
        used = [-(-x // page) for x in lengths]
        pages = sum(used) + 2
        self.cuda, self.bits, self.n, self.h, self.lengths, self.packed, self.causal, self.page = cuda, bits, n, h, lengths, packed, causal, page
        self.k, self.v = (_x(pages, hk, page, d, seed=i) for i in range(2))
        self.table = _table(used, max(max(used), 1), pages)
        self.q = _x(len(lengths), h, n, d, seed=5)

    def pages(self, k):
        """k's pages as the cache holds them, poisoned behind the sequences."""
        return (_poison(_store(x.clone(), self.bits, value), self.table, self.lengths, self.page) for x, value in ((k, False), (self.v, True)))

    def at(self, b, j):
        return int(self.table[b, j // self.page]), j % self.page

    def call(self, k, q):
        kp, vp = (x.to(self.cuda) for x in self.pages(k))
        b, n = len(self.lengths), self.n
        args = (kp, vp, self.table.to(self.cuda), torch.tensor(self.lengths, dtype=torch.int32, device=self.cuda))
        if not self.packed:
            q = q.to(self.cuda)
            return lambda: ktt.sdpa_paged(q, *args, is_causal=self.causal)
        q = q.transpose(1, 2).reshape(b * n, self.h, -1).to(self.cuda)
        cu = torch.arange(b + 1, dtype=torch.int32, device=self.cuda) * n
        return lambda: ktt.sdpa_paged(q, *args, is_causal=self.causal, cu_seq_q=cu, max_q=n)

    def __call__(self, k=None, q=None):
        out = self.call(self.k if k is None else k, self.q if q is None else q)()
        b = len(self.lengths)
        return (out.view(b, self.n, self.h, -1).transpose(1, 2) if self.packed else out).cpu()

    def assert_path(self, cut):
        if cut is None:
            return
        names = [x.name for x in launched(self.call(self.k, self.q))]
        assert any("merge_parts" in name for name in names) == cut and any("fwd_" in name for name in names), names


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("d,h,hk,n,lengths,cut", CASES)
def test_queries(cuda, bits, packed, d, h, hk, n, lengths, cut):
    """A row of NaN and one with an infinity (half of its logits are infinite, of either sign) beside rows that keep their bits."""
    run = _Run(cuda, bits, d, h, hk, n, lengths, packed)
    run.assert_path(cut)
    clean = run()
    assert torch.isfinite(clean).all()
    for x in (NAN, INF):
        q = run.q.clone()
        q[0, 1, n // 2, 3] = x
        got = run(q=q)
        assert got[0, 1, n // 2].isnan().all()
        got[0, 1, n // 2] = clean[0, 1, n // 2]
        assert torch.equal(got, clean)


def _places(n, length):
    """Keys that all rows see: of every eighth of a tile, and further ones."""
    return [j for j in (0, 21, 38, 63, 64, 77, 101, 127, 128, 700, 1500, length - n) if j <= length - n]


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("d,h,hk,n,lengths,cut", CASES)
def test_keys_that_all_rows_see(cuda, bits, packed, d, h, hk, n, lengths, cut):
    """A NaN in a key of one K / V head: none of its query heads' rows has a finite value, all others keep their bits."""
    run = _Run(cuda, bits, d, h, hk, n, lengths, packed)
    clean, group = run(), h // hk
    for j in _places(n, lengths[0]):
        page, row = run.at(0, j)
        k = run.k.clone()
        k[page, 0, row, 5] = NAN
        got = run(k=k)
        assert not torch.isfinite(got[0, :group]).any(), j
        got[0, :group] = clean[0, :group]
        assert torch.equal(got, clean), j


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("d,h,hk,n,lengths,cut", CASES)
def test_an_infinite_key(cuda, packed, d, h, hk, n, lengths, cut):
    """bf16: rows whose query is positive in its column have an infinite logit and nothing finite; to the others the key is not
    there (its logit is -inf)."""
    run = _Run(cuda, 16, d, h, hk, n, lengths, packed)
    group = h // hk
    for j in _places(n, lengths[0])[::3]:
        page, row = run.at(0, j)
        k = run.k.clone()
        k[page, 0, row, 5] = INF
        got = run(k=k)[0, :group]
        up = run.q[0, :group, :, 5] > 0
        assert (run.q[0, :group, :, 5] != 0).all()
        assert not torch.isfinite(got[up]).any() and torch.isfinite(got[~up]).all()
        want, _, _ = po.attend([run.q[0].double()], k, run.v, run.table[:1], lengths[:1], True, d ** -0.5)
        off = (got[~up].double() - want[0][:group][~up]).abs()
        # Half a step of bf16 weights and of the result, of |v| <= 6 (and sums and logits in fp32: less than that once more).
        assert off.max() <= 3 * 2.0 ** -8 * run.v.abs().max()


@pytest.mark.parametrize("kernel,d", [("flash", 64), ("flash_wide", 64), ("flash_wide", 128), ("flash_pair", 64), ("flash_pair", 80), ("flash_pair", 128), ("mma", 64)])
def test_keys_of_the_dense_forward(cuda, kernel, d):
    """The kernels that chunks run on, over plain keys: a NaN at every place of two blocks, a head each."""
    h, n = 256, 256
    q, k, v = (_x(1, h, n, d, seed=i).to(cuda) for i in range(3))
    k[0, torch.arange(h), torch.arange(n), 3] = NAN
    out, _ = ops.sdpa_forward(q, k, v, kernel=kernel)
    assert not torch.isfinite(out).any()
