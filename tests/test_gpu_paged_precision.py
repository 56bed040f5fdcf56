"""How near chunks of prompts over 4-bit pages are to float64: as near as single tokens, whatever the values' magnitude."""

import pytest
import torch

import kohaku_tt_b200 as ktt
from oracle import paged_oracle as po
from tests.launched import launched
from tests.test_gpu_paged import _near, _poison, _table, _x

pytestmark = pytest.mark.gpu


def _attend(cuda, d, h, hk, n, lengths, packed, causal, values, cut=None, keys=lambda i, j: 1.0, queries=1.0):
    """(outputs, oracle's) of queries over a cache; `values`, `keys`: factors of those, by the sequence and the key."""
    page, b = 32, len(lengths)
    used = [-(-x // page) for x in lengths]
    pages = sum(used) + 1
    table = _table(used, max(used), pages)
    k, v = (_x(pages, hk, page, d, seed=i) for i in range(2))
    for i, length in enumerate(lengths):
        for j in range(length):
            v[int(table[i, j // page]), :, j % page] *= values(i, j)
            k[int(table[i, j // page]), :, j % page] *= keys(i, j)
    kp, vp = _poison(po.pack(k, False), table, lengths, page), _poison(po.pack(v, True), table, lengths, page)
    q = _x(b, h, n, d, seed=9) * queries
    want, mags, sizes = po.attend([x.double() for x in q], kp, vp, table, lengths, causal, d ** -0.5)
    args = (kp.to(cuda), vp.to(cuda), table.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda))
    kw = dict(is_causal=causal)
    qd = q.to(cuda)
    if packed:
        qd, kw["cu_seq_q"], kw["max_q"] = qd.transpose(1, 2).reshape(b * n, h, d), torch.arange(b + 1, dtype=torch.int32, device=cuda) * n, n
    if cut is not None:
        assert any("merge_parts" in x.name for x in launched(lambda: ktt.sdpa_paged(qd, *args, **kw))) == cut
    out = ktt.sdpa_paged(qd, *args, **kw)
    return list(out.view(b, n, h, d).transpose(1, 2) if packed else out), want, mags, sizes


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d,h,hk,n,lengths,cut", [(128, 2, 1, 130, [3000, 1025], True), (64, 2, 1, 130, [3000, 1025], True), (128, 8, 2, 130, [600, 457], False),
                                                  (64, 8, 2, 130, [600, 457], False), (128, 8, 2, 4, [600, 457], None), (64, 8, 2, 4, [600, 457], None)])
def test_roundings(cuda, packed, causal, d, h, hk, n, lengths, cut):
    """Root mean squares against that of the result's own rounding to bf16. In chunks nothing else is rounded to as few bits, and three
    roundings to fp16 (queries, which are exact there, left out) are an eighth each: sqrt(1 + 3 / 64) = 1.02. The pass over a few tokens
    rounds its weights to bf16: about as much again, with signs of their own, sqrt(2). 1.2 and 1.6 leave one more of bf16's errors out."""
    got, want, _, _ = _attend(cuda, d, h, hk, n, lengths, packed, causal, lambda i, j: 1.0, cut)
    got, want = torch.stack(got).double().cpu(), torch.stack(want)
    own = (want.to(torch.bfloat16).double() - want).pow(2).mean().sqrt()
    assert (got - want).pow(2).mean().sqrt() <= (1.6 if n == 4 else 1.2) * own


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("d,h,hk,n,lengths,cut", [(128, 2, 1, 130, [3000, 1025], True), (64, 2, 1, 130, [3000, 1025], True), (128, 8, 2, 130, [600, 457], False),
                                                  (64, 8, 2, 130, [600, 457], False)])
def test_magnitudes(cuda, packed, d, h, hk, n, lengths, cut):
    """Values that are large or small as a whole, change from one group of 64 keys to the next, or are zero."""
    steps = [0, 40, -40, 12, 0, -3, 55, -55, 1, 20]
    for values in (lambda i, j: 2.0 ** 100, lambda i, j: 2.0 ** -60, lambda i, j: 2.0 ** steps[j // 64 % 10], lambda i, j: 2.0 ** steps[j * 7 % 10],
                   lambda i, j: 0.0 if i else 2.0 ** -j, lambda i, j: 0.0 if j % 128 < 64 else 1.0):
        got, want, mags, sizes = _attend(cuda, d, h, hk, n, lengths, packed, True, values, cut)
        _near(got, want, mags, sizes, True)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("d,h,hk,n,lengths,cut", [(128, 2, 1, 130, [3000, 1025], True), (64, 2, 1, 130, [3000, 1025], True), (128, 8, 2, 130, [600, 457], False),
                                                  (64, 8, 2, 130, [600, 457], False)])
def test_magnitudes_of_queries_and_keys(cuda, packed, d, h, hk, n, lengths, cut):
    """Far from 1 in opposite directions; keys that change from one group of 64 to the next, are small, or zero; rows of queries apart."""
    rows = 2.0 ** torch.arange(-n // 2, n - n // 2).clamp(-60, 0).to(torch.bfloat16)[:, None]
    for keys, queries in ((lambda i, j: 2.0 ** -60, 2.0 ** 60), (lambda i, j: 2.0 ** 60, 2.0 ** -60), (lambda i, j: 2.0 ** -(j // 64 % 7), 1.0),
                          (lambda i, j: 0.0 if j % 128 < 64 else 1.0, 1.0), (lambda i, j: 2.0 ** -j, 1.0), (lambda i, j: 1.0, rows)):
        got, want, mags, sizes = _attend(cuda, d, h, hk, n, lengths, packed, True, lambda i, j: 1.0, cut, keys, queries)
        _near(got, want, mags, sizes, True)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [4, 130])
@pytest.mark.parametrize("x", [float("nan"), float("inf"), float("-inf")])
def test_a_value_that_is_no_number(cuda, d, n, x):
    """It shows in the channels of its group of 64, and in no other."""
    lengths = [600, 300]

    def values(i, j):
        by = torch.ones(d, dtype=torch.bfloat16)
        if i == 0 and j == 100:
            by[3] = x
        return by

    got, want, mags, sizes = _attend(cuda, d, 8, 2, n, lengths, False, True, values)
    assert not torch.isfinite(got[0][..., :64]).any()
    _near([got[1]] + ([got[0][..., 64:]] if d == 128 else []), [want[1]] + ([want[0][..., 64:]] if d == 128 else []),
          [mags[1]] + ([mags[0][..., 64:]] if d == 128 else []), [sizes[1]] + ([sizes[0]] if d == 128 else []), True)
