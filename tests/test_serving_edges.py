"""What the entries of a server's steps refuse where they are not plain, without a GPU (no kernel is launched in this file)."""

import ctypes

import torch

from kohaku_tt_b200 import _lib
from oracle import serving_oracle as so


def _append(**kw):
    x = _lib.AppendAtArgs()
    a = x.base
    c = a.cache
    c.k = c.v = c.block_table = c.lengths = 4096
    c.bits, c.page_size, c.kv_heads, c.table_width, c.pages, c.table_stride = 16, 16, 2, 4, 9, 4
    for f in (c.k_strides, c.v_strides):
        f[0], f[1], f[2] = 2048, 1024, 64
    a.batch, a.rows, a.d, a.k, a.v = 2, 1, 64, 4096, 4096
    for name, v in kw.items():
        setattr(a, name, v)
    return x


def test_granted_refusals(built_lib):
    for out in (8192, 8188, 8196):      # two words each: on one another in part or whole
        assert built_lib.ktt_b200_paged_append_granted(ctypes.byref(_append(lengths_out=out)), 8192, None) == _lib.ERR_BAD_ARGUMENT
        assert "granted" in _lib.last_error()
    assert built_lib.ktt_b200_paged_append_granted(ctypes.byref(_append(rows=0)), 8192, None) == 0      # nothing to do
    assert built_lib.ktt_b200_paged_append_granted(ctypes.byref(_append(k=None)), 8192, None) == _lib.ERR_BAD_ARGUMENT
    assert built_lib.ktt_b200_paged_append_granted(None, 8192, None) == _lib.ERR_BAD_ARGUMENT


def test_append_by_hand():
    """Of 3 rows behind 15 keys the first two go in, one to each page; a sequence that got nothing stays as it is."""
    pages = torch.zeros((3, 1, 16, 1))
    rows = [torch.tensor([1.0, 2.0, 3.0]).view(3, 1, 1), torch.tensor([4.0]).view(1, 1, 1)]
    assert so.append(pages, torch.tensor([[2, 0], [1, -1]]), [15, 3], rows, [2, 0]) == [17, 3]
    assert pages[2, 0, 15] == 1 and pages[0, 0, 0] == 2 and pages.abs().sum() == 3


def _tables(**kw):
    a = _lib.Tables()
    a.batch, a.table_width, a.page_size, a.table_stride, a.pool = 2, 4, 16, 4, 8
    a.block_table = a.lengths = a.free_pages = a.count = 4096
    a.count_out = 8192
    for name, x in kw.items():
        setattr(a, name, x)
    return a


def _bounds(strides=(256, 128, 64), **kw):
    b = _lib.BoundsArgs(cache=_append().base.cache)
    b.batch, b.d, b.bounds = 2, 64, 4096
    for i, x in enumerate(strides):
        b.bounds_strides[i] = x
    for name, x in kw.items():
        setattr(b if name in ("batch", "d", "bounds") else b.cache, name, x)
    return b


def test_release_with_bounds_refusals(built_lib):
    """What is not of the same table is refused, and so is what either half refuses."""
    for kw in (dict(batch=1), dict(page_size=32), dict(table_width=3), dict(block_table=8192), dict(lengths=8192), dict(table_stride=5), dict(max_keys=32)):
        assert built_lib.ktt_b200_paged_release_bounds(ctypes.byref(_tables()), 4096, ctypes.byref(_bounds(**kw)), None) == _lib.ERR_BAD_ARGUMENT, kw
        assert "same table" in _lib.last_error()
    for kw, status in ((dict(bounds=None), _lib.ERR_BAD_ARGUMENT), (dict(bounds=4104), _lib.ERR_UNSUPPORTED), (dict(d=96), _lib.ERR_UNSUPPORTED), (dict(strides=(0, 128, 64)), _lib.ERR_UNSUPPORTED)):
        assert built_lib.ktt_b200_paged_release_bounds(ctypes.byref(_tables()), 4096, ctypes.byref(_bounds(**kw)), None) == status
    for kw, status in ((dict(batch=4097), _lib.ERR_UNSUPPORTED), (dict(count_out=4096), _lib.ERR_BAD_ARGUMENT)):
        assert built_lib.ktt_b200_paged_release_bounds(ctypes.byref(_tables(**kw)), 4096, ctypes.byref(_bounds()), None) == status
    assert built_lib.ktt_b200_paged_release_bounds(ctypes.byref(_tables()), None, ctypes.byref(_bounds()), None) == _lib.ERR_BAD_ARGUMENT
    assert built_lib.ktt_b200_paged_release_bounds(None, 4096, ctypes.byref(_bounds()), None) == _lib.ERR_BAD_ARGUMENT
