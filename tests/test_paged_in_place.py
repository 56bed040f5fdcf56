"""The C entries of rotary positions and the paged cache refuse an output that is its input (no kernel is launched in this file)."""

import ctypes

import pytest

from kohaku_tt_b200 import _lib


def _pages(c):
    c.k = c.v = c.block_table = c.lengths = 4096
    c.bits, c.page_size, c.kv_heads, c.table_width, c.pages, c.table_stride = 16, 16, 2, 4, 9, 4
    for f in (c.k_strides, c.v_strides):
        f[0], f[1], f[2] = 4096, 2048, 128


@pytest.mark.parametrize("name", ["q", "k"])
def test_rotary(built_lib, name):
    a = _lib.RotaryArgs()
    a.batch, a.rows, a.heads, a.kv_heads, a.d, a.pairs, a.dtype, a.table_rows = 1, 1, 1, 1, 64, 32, _lib.MASK_BF16, 4
    a.q, a.q_out, a.k, a.k_out, a.cos, a.sin = 4096, 8192, 16384, 32768, 65536, 65536
    setattr(a, name + "_out", getattr(a, name))
    assert built_lib.ktt_b200_rotary(ctypes.byref(a), None) == _lib.ERR_BAD_ARGUMENT and "overlap" in _lib.last_error()


def test_append(built_lib):
    a = _lib.AppendArgs()
    _pages(a.cache)
    a.batch, a.rows, a.d, a.heads, a.k, a.v, a.q, a.q_out = 1, 1, 128, 2, 4096, 4096, 8192, 8192
    assert built_lib.ktt_b200_paged_append(ctypes.byref(a), None) == _lib.ERR_BAD_ARGUMENT and "overlap" in _lib.last_error()


@pytest.mark.parametrize("sq", [1, 200])
def test_attention(built_lib, sq):
    a = _lib.PagedSdpaArgs()
    _pages(a.cache)
    a.batch, a.heads, a.sq, a.d, a.scale, a.q, a.out, a.workspace, a.workspace_bytes = 1, 4, sq, 128, 0.1, 4096, 4096, 4096, 1 << 40
    assert built_lib.ktt_b200_paged_sdpa(ctypes.byref(a), None) == _lib.ERR_BAD_ARGUMENT and "overlap" in _lib.last_error()
