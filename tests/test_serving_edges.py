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
