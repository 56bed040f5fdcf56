"""Sequences without a key: zeros, whatever their queries hold and whichever way a call takes."""

import pytest
import torch

from tests.test_gpu_paged_nan import INF, NAN, _Run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d,h,hk,n,lengths,cut", [
    (128, 2, 1, 130, [0, 3000, 0], True), (64, 2, 1, 130, [0, 3000, 0], True), (128, 8, 2, 130, [0, 300, 0], False), (64, 8, 2, 130, [0, 300, 0], False),
    (128, 4, 2, 70, [0, 0, 0], False), (64, 4, 2, 70, [0, 0, 0], False), (128, 16, 2, 4, [0, 300, 0], None), (64, 14, 2, 1, [0, 9000, 0], None)])
def test_queries_without_keys(cuda, bits, packed, causal, d, h, hk, n, lengths, cut):
    run = _Run(cuda, bits, d, h, hk, n, lengths, packed, causal)
    run.assert_path(cut)
    clean = run()
    q = run.q.clone()
    q[0], q[2] = NAN, INF
    got = run(q=q)
    assert not got[0].any() and not got[2].any()
    assert torch.equal(got[1], clean[1])
