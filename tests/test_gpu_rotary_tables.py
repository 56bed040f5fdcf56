"""What scaled tables are off by, and tables made inside of compiled and traced code."""

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


def test_compiled(cuda):
    x = torch.randn((1, 2, 16, 64), device=cuda).bfloat16()
    how = dict(base=1e6, scaling="parts", factor=4.0, original=8)

    def turned(x):
        cos, sin = ktt.rotary_table(16, 64, device=x.device, **how)
        return ktt.rotary(x, None, cos, sin)[0], cos, sin

    want = turned(x)
    for a, b in zip(torch.compile(turned, fullgraph=True)(x), want):
        assert torch.equal(a, b)


def test_fake_tables_are_fake(cuda):
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode

    for device in ("cuda", cuda):
        with FakeTensorMode():
            cos, sin = ktt.rotary_table(16, 64, device=device)
        for t in (cos, sin):
            assert isinstance(t, FakeTensor) and t.shape == (16, 32) and t.dtype == torch.float32 and t.device == cuda


def test_modes_that_watch_calls(cuda):
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    class Functions(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    seen = []

    class Operators(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    want = ktt.rotary_table(16, 64, device=cuda)
    for mode in (Functions(), Operators()):
        with mode:
            got = ktt.rotary_table(16, 64, device=cuda)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert any("_rotary_table" in name for name in seen)
    for bad in (dict(positions=0, dim=64), dict(positions=4, dim=63), dict(positions=4, dim=514), dict(positions=4, dim=64, scaling="parts", factor=2.0)):
        with Operators(), pytest.raises(ValueError):
            ktt.rotary_table(**bad)
