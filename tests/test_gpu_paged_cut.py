"""Packed chunks that are cut along their keys, where the launches of a call share the packed rows and where a buffer has more rows
than its sequences, against float64."""

import pytest
import torch

import kohaku_tt_b200 as ktt
from oracle import paged_oracle as po
from tests.launched import launched
from tests.test_gpu_paged import _cache, _near, _x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d,h,hk,counts,lengths,wide,rows", [
    (128, 8, 8, [130, 60, 7, 129], [3000, 100, 0, 2049], 2048, 326),    # 131,072 places, so two launches of two sequences
    (64, 16, 16, [130, 60, 7, 129], [3000, 100, 0, 2049], 2048, 326),
    (128, 8, 8, [100], [3000], 47, 900), (64, 8, 2, [100], [3000], 47, 900),
    (128, 2, 1, [130, 3], [3000, 1100], 47, 1000), (64, 2, 1, [130, 3], [3000, 1100], 47, 133)])
def test_packed(cuda, bits, d, h, hk, counts, lengths, wide, rows):
    kp, vp, table = _cache(bits, d, hk, 64, lengths, wide=wide)
    qs = [_x(h, n, d, seed=10 + i) for i, n in enumerate(counts)]
    q = torch.full((rows, h, d), float("nan"), dtype=torch.bfloat16)
    q[:sum(counts)] = torch.cat([x.transpose(0, 1) for x in qs])
    cu = torch.tensor([0] + counts).cumsum(0).to(device=cuda, dtype=torch.int32)
    args = (q.to(cuda), kp.to(cuda), vp.to(cuda), table.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda))
    names = [x.name for x in launched(lambda: ktt.sdpa_paged(*args, cu_seq_q=cu, max_q=max(counts)))]
    assert sum("merge_parts" in name for name in names) == (2 if len(counts) == 4 else 1), names
    out = ktt.sdpa_paged(*args, cu_seq_q=cu, max_q=max(counts))
    got = [out[cu[i]:cu[i + 1]].transpose(0, 1) for i in range(len(counts))]
    want, mags, sizes = po.attend([x.double() for x in qs], kp.nan_to_num(0.0) if bits == 16 else kp, vp.nan_to_num(0.0) if bits == 16 else vp, table, lengths, True, d ** -0.5)
    _near(got, want, mags, sizes, bits == 4)
