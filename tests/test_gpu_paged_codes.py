"""Codes of groups whose steps are subnormal: a step of a few of the least bf16 values is rounded by as much as half of one, and
the farthest values then lie past 15 of them."""

import pytest
import torch

import kohaku_tt_b200 as ktt
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu

LEAST = 2.0 ** -133     # of the bf16 values above 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("least", [0.0, -7 * LEAST, -100 * LEAST])
def test_ranges_of_a_few_of_the_least_values(cuda, d, least):
    """Ranges of 1 to 255 of them: codes, steps and least values to the bit, 0 to 15 of them."""
    n = 256
    part = torch.rand((n, 1, d), generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    part[..., 0::64], part[..., 1::64] = 0.0, 1.0
    whole = torch.arange(n, dtype=torch.float64)[:, None, None]
    x = (least + torch.round(part * whole) * LEAST).to(torch.bfloat16)
    kp, vp = ktt.paged_cache(n // 16, 1, 16, d, bits=4, device=cuda)
    table = torch.arange(n // 16, dtype=torch.int32, device=cuda)[None]
    xd = x.transpose(0, 1)[None].to(cuda)
    ktt.paged_append(xd, xd, kp, vp, table, torch.zeros(1, dtype=torch.int32, device=cuda))
    want = po.quantise(x)
    assert (want[0].max() == 15) and (want[1] > 0).any()
    for pages, value in ((kp, False), (vp, True)):
        got = po.unpack(pages.cpu(), value)
        for a, b in zip(got, want):
            assert torch.equal(a.transpose(1, 2).reshape(b.shape), b)
