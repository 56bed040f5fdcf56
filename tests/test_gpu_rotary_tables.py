"""What scaled tables are off by."""

import pytest
import torch

import kohaku_tt_b200 as ktt
from kohaku_tt_b200.rotary import rotary_frequencies
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("positions", [2048, 32768])
@pytest.mark.parametrize("factor", [2.3125, 3.0625, 1.1875])
def test_the_scale_is_not_rounded_before_the_entries_are(cuda, positions, factor):
    """These factors' scales are 0.87 to 0.91 x 2^-24 of themselves away from fp32's next. As a factor of every entry that would
    be there in the slope of entries over their values; what roundings by themselves leave of it is the root of their
    number less: each of 65,536 entries at least is off by 2^-23 at most where the mean of the squares is 1/2 and more, that is
    2^-23 / sqrt(32768) = 2^-30.5 (one standard error). Eight of them: 2^-27.5, an eleventh of what is looked for."""
    cos, sin = ktt.rotary_table(positions, 64, scaling="parts", factor=factor, original=1024, device=cuda)
    f, scale = rotary_frequencies(64, scaling="parts", factor=factor, original=1024)
    step = torch.tensor(scale, dtype=torch.float32).double().item() / scale - 1
    assert abs(step) > 0.85 * 2.0 ** -24
    want = torch.stack(po.table(positions, f, scale))
    off = torch.stack([cos, sin]).double().cpu() - want
    assert abs((off * want).sum() / (want * want).sum()) <= 2.0 ** -27.5
