"""Layouts of results where operands lie apart: those that compiled graphs are told are those that the operators give."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import kohaku_tt_b200 as ktt
from tests.test_gpu_paged import _x

pytestmark = pytest.mark.gpu

H, HK, N, D = 4, 2, 5, 64


def _columns_apart(heads):
    return _x(2, D, heads, N, seed=heads).permute(0, 2, 3, 1)


def _every_other_column(heads):
    return _x(2, N, heads, 2 * D, seed=heads).transpose(1, 2)[..., ::2]


def _unaligned_heads(heads):
    return _x(2, N, heads * D + 8, seed=heads)[..., 1:heads * D + 1].unflatten(-1, (heads, D)).transpose(1, 2)


def _heads(heads):
    return _x(2, N, heads * D, seed=heads).unflatten(-1, (heads, D)).transpose(1, 2)


def _expanded(heads):
    return _x(2, 1, N, D, seed=heads).expand(2, heads, N, D)


LAYOUTS = [_columns_apart, _every_other_column, _unaligned_heads, _heads, _expanded]


def _calls(cuda):
    kp, vp = (_x(8, HK, 16, D, seed=i).to(cuda) for i in range(2))
    table = torch.arange(8, dtype=torch.int32, device=cuda).view(2, 4)
    lens = torch.tensor([20, 33], dtype=torch.int32, device=cuda)
    cos, sin = ktt.rotary_table(64, D, device=cuda)
    ops = torch.ops.ktt_b200
    return {
        "rotary": (lambda q, k, *rest: ops._rotary(q, k, *rest, None, False, False), lambda q, k, *rest: ktt.rotary(q, k, *rest), (cos, sin)),
        "append": (lambda q, k, kp, vp, t, l, c, s: ops._paged_append(k, k, kp, vp, t, l, c, s, q, False, None, None),
                   lambda q, k, kp, vp, t, l, c, s: ktt.paged_append(k, k, kp, vp, t, l, c, s, q=q), (kp, vp, table, lens, cos, sin)),
        "attend": (lambda q, k, *rest: ops._sdpa_paged(q, *rest, True, None, None, None, None), lambda q, k, *rest: ktt.sdpa_paged(q, *rest), (kp, vp, table, lens)),
    }


def _moved(t, cuda):
    """t on the device, in the same places of its storage."""
    base = torch.empty(t.untyped_storage().nbytes() // 2, dtype=t.dtype)
    base.set_(t.untyped_storage(), 0, base.shape)
    return torch.as_strided(base.to(cuda), t.shape, t.stride(), t.storage_offset())


def _list(out):
    return list(out) if isinstance(out, (tuple, list)) else [out]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("name", ["rotary", "append", "attend"])
def test_layouts_of_results(cuda, name, layout):
    op, call, rest = _calls(cuda)[name]
    q, k = (_moved(layout(heads), cuda) for heads in (H, HK))
    real = _list(op(q, k, *rest))
    eager = _list(call(q, k, *rest))
    with FakeTensorMode(allow_non_fake_inputs=False) as mode:
        fake = _list(op(*[mode.from_tensor(t) for t in (q, k, *rest)]))
    assert [t.stride() for t in fake] == [t.stride() for t in real] == [t.stride() for t in eager]
    compiled = _list(torch.compile(call, fullgraph=True)(q, k, *rest))
    assert [t.stride() for t in compiled] == [t.stride() for t in eager]
    for a, b, c in zip(real, eager, compiled):
        assert torch.equal(a, b) and torch.equal(a, c)
