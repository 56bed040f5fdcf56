"""Block tables, positions of several axes, bounds and selected pages without a GPU: what the entries refuse (no kernel is
launched in this file), and the oracle's own sums."""

import ctypes

import pytest
import torch

import kohaku_tt_b200 as ktt
from kohaku_tt_b200 import _lib
from kohaku_tt_b200.rotary import check_positions, pair_axes, position_strides
from oracle import serving_oracle as so


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_tables_by_hand():
    table, cu, positions, slots, granted, left = so.reserve([[7, -1, -1], [-1, -1, -1], [4, 5, -1]], [10, 0, 32], [7, 3, 1], [9, 8, 3, 2], 4, 16, 12)
    assert table == [[7, 2, -1], [3, -1, -1], [4, 5, 8]] and cu == [0, 7, 10, 11] and left == 1 and granted == [7, 3, 1]
    assert positions == [10, 11, 12, 13, 14, 15, 16, 0, 1, 2, 32, -1]
    assert slots == [7 * 16 + 10 + i for i in range(6)] + [2 * 16, 3 * 16, 3 * 16 + 1, 3 * 16 + 2, 8 * 16, -1]
    assert so.reserve([[7, -1], [-1, -1], [1, -1]], [10, 0, 3], [7, 3, 2], [9], 1, 16, 12)[4:] == ([7, 0, 0], 0)      # those behind get none either
    assert so.release(table, [17, 3, 33], [10, 0, 33], [9, 8, 3, 2], 1, 16) == ([[7, -1, -1], [-1, -1, -1], [4, 5, 8]], [9, 2, 3, 2], 3)


def _tables(**kw):
    a = _lib.Tables()
    a.batch, a.table_width, a.page_size, a.table_stride, a.pool = 2, 4, 16, 4, 8
    a.block_table = a.lengths = a.free_pages = a.count = 4096
    a.count_out = 8192
    for name, x in kw.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("kw,status,text", [
    (dict(batch=0), _lib.ERR_UNSUPPORTED, "positive"), (dict(table_width=0), _lib.ERR_UNSUPPORTED, "positive"), (dict(page_size=24), _lib.ERR_UNSUPPORTED, "multiple of 16"),
    (dict(page_size=0), _lib.ERR_UNSUPPORTED, "multiple of 16"), (dict(batch=4097), _lib.ERR_UNSUPPORTED, "4096"), (dict(table_width=1 << 27), _lib.ERR_UNSUPPORTED, "2^30"),
    (dict(table_stride=3), _lib.ERR_UNSUPPORTED, "on one another"), (dict(table_stride=0), _lib.ERR_UNSUPPORTED, "on one another"),
    (dict(table_stride=-3), _lib.ERR_UNSUPPORTED, "on one another"), (dict(pool=1 << 31), _lib.ERR_UNSUPPORTED, "2^31"), (dict(pool=-1), _lib.ERR_UNSUPPORTED, "positive"), (dict(count=None), _lib.ERR_BAD_ARGUMENT, "null"),
    (dict(count_out=4096), _lib.ERR_BAD_ARGUMENT, "another word"), (dict(free_pages=None), _lib.ERR_BAD_ARGUMENT, "null"), (dict(block_table=None), _lib.ERR_BAD_ARGUMENT, "null")])
def test_tables_that_no_entry_takes(built_lib, kw, status, text):
    assert built_lib.ktt_b200_paged_reserve(ctypes.byref(_tables(**kw)), 4096, 3, None, None, None, None, None) == status
    assert text in _lib.last_error()
    assert built_lib.ktt_b200_paged_release(ctypes.byref(_tables(**kw)), 4096, None) == status
    assert text in _lib.last_error()


def test_reserve_and_release_refusals(built_lib):
    for tokens in (-1, 1 << 31):
        assert built_lib.ktt_b200_paged_reserve(ctypes.byref(_tables()), 4096, tokens, None, None, None, None, None) == _lib.ERR_BAD_ARGUMENT
    assert built_lib.ktt_b200_paged_reserve(ctypes.byref(_tables()), None, 1, None, None, None, None, None) == _lib.ERR_BAD_ARGUMENT
    assert built_lib.ktt_b200_paged_release(ctypes.byref(_tables()), None, None) == _lib.ERR_BAD_ARGUMENT
    assert built_lib.ktt_b200_paged_reserve(None, 4096, 1, None, None, None, None, None) == _lib.ERR_BAD_ARGUMENT
    assert built_lib.ktt_b200_paged_release(None, 4096, None) == _lib.ERR_BAD_ARGUMENT


def _pages(**kw):
    c = _lib.Pages()
    c.k = c.v = c.block_table = c.lengths = 4096
    c.bits, c.page_size, c.kv_heads, c.table_width, c.pages = 16, 16, 2, 4, 9
    for f in (c.k_strides, c.v_strides):
        f[0], f[1], f[2] = 4096, 2048, 128
    c.table_stride = 4
    for name, x in kw.items():
        setattr(c, name, x)
    return c


def _axes(of_pair=bytes([0, 1]), **kw):
    x = _lib.Axes()
    x.axes, x.positions, x.of_pair = 2, 4096, of_pair
    for name, v in kw.items():
        setattr(x, name, v)
    return x


def test_axes_refusals(built_lib):
    a = _lib.RotaryArgs()
    a.batch = a.rows = a.heads = 1
    a.d, a.pairs, a.dtype, a.q, a.q_out, a.cos, a.sin, a.table_rows = 8, 2, _lib.MASK_BF16, 4096, 8192, 4096, 4096, 4
    for x, text in ((_axes(axes=0), "1 to 4"), (_axes(axes=5), "1 to 4"), (_axes(positions=None), "null"), (_axes(of_pair=None), "null"),
                    (_axes(of_pair=bytes([0, 2])), "one of the positions")):
        assert built_lib.ktt_b200_rotary_axes(ctypes.byref(a), ctypes.byref(x), None) == _lib.ERR_BAD_ARGUMENT
        assert text in _lib.last_error()
        append = _lib.AppendAtArgs(base=_lib.AppendArgs(cache=_pages()), positions=x)
        b = append.base
        b.batch, b.rows, b.d, b.k, b.v, b.cos, b.sin, b.pairs, b.table_rows = 1, 1, 64, 4096, 4096, 4096, 4096, 2, 4
        status = built_lib.ktt_b200_paged_append_at(ctypes.byref(append), None)
        if x.positions:   # (none: rows turn by their places)
            assert status == _lib.ERR_BAD_ARGUMENT and text in _lib.last_error()
    assert built_lib.ktt_b200_rotary_axes(ctypes.byref(a), None, None) == _lib.ERR_BAD_ARGUMENT
    assert built_lib.ktt_b200_rotary_axes(None, ctypes.byref(_axes()), None) == _lib.ERR_BAD_ARGUMENT
    a.pairs = 5
    assert built_lib.ktt_b200_rotary_axes(ctypes.byref(a), ctypes.byref(_axes()), None) == _lib.ERR_BAD_ARGUMENT
    assert built_lib.ktt_b200_paged_append_at(None, None) == _lib.ERR_BAD_ARGUMENT


def test_bounds_refusals(built_lib):
    def args(strides=(512, 256, 128), bounds=4096, **kw):
        a = _lib.BoundsArgs(cache=_pages())
        a.batch, a.d, a.bounds = 1, 128, bounds
        for i, x in enumerate(strides):
            a.bounds_strides[i] = x
        for name, x in kw.items():
            setattr(a, name, x)
        return a

    for a, status in ((args(bounds=4104), _lib.ERR_UNSUPPORTED), (args(strides=(512, 256, 100)), _lib.ERR_UNSUPPORTED),
                      (args(strides=(0, 256, 128)), _lib.ERR_UNSUPPORTED), (args(strides=(512, 64, 128)), _lib.ERR_UNSUPPORTED), (args(strides=(512, 256, 0)), _lib.ERR_UNSUPPORTED), (args(d=96), _lib.ERR_UNSUPPORTED),
                      (args(batch=65536), _lib.ERR_UNSUPPORTED), (args(batch=0), _lib.ERR_BAD_ARGUMENT), (args(bounds=None), _lib.ERR_BAD_ARGUMENT)):
        assert built_lib.ktt_b200_paged_bounds(ctypes.byref(a), None) == status
    assert built_lib.ktt_b200_paged_bounds(None, None) == _lib.ERR_BAD_ARGUMENT
    append = _lib.AppendAtArgs(base=_lib.AppendArgs(cache=_pages()), bounds=4104)
    append.base.batch, append.base.rows, append.base.d, append.base.k, append.base.v = 1, 1, 64, 4096, 4096
    assert built_lib.ktt_b200_paged_append_at(ctypes.byref(append), None) == _lib.ERR_UNSUPPORTED
    append.base.k = None
    assert built_lib.ktt_b200_paged_append_at(ctypes.byref(append), None) == _lib.ERR_BAD_ARGUMENT


def _select(**kw):
    a = _lib.SelectArgs()
    a.batch, a.heads, a.kv_heads, a.sq, a.d, a.page_size, a.table_width, a.pages, a.table_stride = 2, 8, 2, 1, 128, 16, 40, 99, 40
    a.top, a.first, a.last = 8, 1, 1
    a.q = a.bounds = a.block_table = a.lengths = a.chosen = a.keys = a.workspace = 4096
    for i, x in enumerate((1024, 128, 128)):
        a.q_strides[i] = x
    for i, x in enumerate((512, 256, 128)):
        a.bounds_strides[i] = x
    for name, x in kw.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("kw,text", [
    (dict(d=96), "head dim"), (dict(page_size=8), "multiple of 16"), (dict(heads=7), "divide"), (dict(top=1), "no more than"), (dict(last=0), "1 or more last"),
    (dict(first=-1), "0 or more first"), (dict(first=8), "no more than"), (dict(first=2 ** 31 - 1, last=2 ** 31 - 1), "no more than"), (dict(table_width=0), "positive"),
    (dict(table_width=(1 << 18) + 1), "262144"), (dict(page_size=1 << 20, table_width=1 << 11), "2^30"), (dict(q=4098), "aligned"), (dict(kv_heads=0), "positive"),
    (dict(batch=65536), "65535"), (dict(top=1 << 19), "no more than")])
def test_selections_that_no_entry_takes(built_lib, kw, text):
    assert built_lib.ktt_b200_paged_select_workspace(ctypes.byref(_select(**kw))) == -1 and text in _lib.last_error()
    assert built_lib.ktt_b200_paged_select(ctypes.byref(_select(**kw)), None) == _lib.ERR_UNSUPPORTED and text in _lib.last_error()


def test_select_refusals(built_lib):
    assert built_lib.ktt_b200_paged_select_workspace(ctypes.byref(_select())) == 0
    wide = dict(table_width=9000, table_stride=9000)      # scores that do not fit shared memory
    need = built_lib.ktt_b200_paged_select_workspace(ctypes.byref(_select(**wide)))
    assert need > 0
    for kw in (dict(batch=0), dict(sq=-1), dict(q=None), dict(bounds=None), dict(chosen=None), dict(keys=None), dict(workspace=None, workspace_bytes=need, **wide),
               dict(workspace_bytes=need - 1, **wide), dict(workspace=4104, workspace_bytes=need, **wide)):
        assert built_lib.ktt_b200_paged_select(ctypes.byref(_select(**kw)), None) == _lib.ERR_BAD_ARGUMENT, kw
    a = _select(workspace_bytes=need)
    a.bounds_strides[0] = 4
    assert built_lib.ktt_b200_paged_select(ctypes.byref(a), None) == _lib.ERR_UNSUPPORTED
    a = _select()
    a.q_strides[1] = 4
    assert built_lib.ktt_b200_paged_select(ctypes.byref(a), None) == _lib.ERR_UNSUPPORTED
    assert built_lib.ktt_b200_paged_select(ctypes.byref(_select(sq=0)), None) == 0      # nothing to do
    assert built_lib.ktt_b200_paged_select(None, None) == _lib.ERR_BAD_ARGUMENT and built_lib.ktt_b200_paged_select_workspace(None) == -1


def test_attention_over_tables_of_tokens_refusals(built_lib):
    def args(**kw):
        a = _lib.PagedSdpaArgs(cache=_pages())
        a.batch, a.heads, a.sq, a.d, a.scale, a.q, a.out, a.workspace = 2, 8, 3, 128, 0.1, 4096, 8192, 4096
        for name, x in kw.items():
            setattr(a, name, x)
        return a

    need = built_lib.ktt_b200_paged_sdpa_chosen_workspace(ctypes.byref(args()))
    assert need > 0
    for kw, text in ((dict(heads=7), "divide"), (dict(scale=0.0), "scale"), (dict(cu_seqlens_q=4096), "one batch entry"), (dict(batch=65535, sq=1 << 20), "2^28"), (dict(d=32), "head dim")):
        assert built_lib.ktt_b200_paged_sdpa_chosen_workspace(ctypes.byref(args(**kw))) == -1 and text in _lib.last_error()
        assert built_lib.ktt_b200_paged_sdpa_chosen(ctypes.byref(args(**kw)), None) == _lib.ERR_UNSUPPORTED and text in _lib.last_error()
    for kw in (dict(batch=0), dict(q=None), dict(out=4096), dict(workspace=None, workspace_bytes=need), dict(workspace_bytes=need - 1)):
        assert built_lib.ktt_b200_paged_sdpa_chosen(ctypes.byref(args(**kw)), None) == _lib.ERR_BAD_ARGUMENT, kw
    assert built_lib.ktt_b200_paged_sdpa_chosen(ctypes.byref(args(sq=0)), None) == 0
    assert built_lib.ktt_b200_paged_sdpa_chosen(None, None) == _lib.ERR_BAD_ARGUMENT


def test_axes_of_pairs():
    assert pair_axes(None, 4, "rotary") is None and pair_axes([0, 1, 2, 3], 4, "rotary") == (0, 1, 2, 3)
    for axes in ((0, 1, 2), (0, 1, 2, 4), (0, 0, 0, -1)):
        with pytest.raises(ValueError, match="axes must name"):
            pair_axes(axes, 4, "rotary")
    q = torch.zeros(2, 3, 5, 8)
    for shape, axes in (((3, 5), (0, 2)), ((3, 2, 5), (0, 2)), ((4, 1, 5), (0, 1)), ((5,), None), ((1, 5), None)):
        check_positions(torch.zeros(shape, dtype=torch.int32), axes, q, 5, "rotary")
    for shape, axes in (((2, 5), (0, 2)), ((3, 4), (0, 2)), ((5, 5), (0, 1)), ((3, 3, 5), (0, 1)), ((5,), (0,)), ((3, 5), None), ((), (0,))):
        with pytest.raises(ValueError, match="positions must have|one position per row"):
            check_positions(torch.zeros(shape, dtype=torch.int32), axes, q, 5, "rotary")
    # (axis, batch, row) strides
    p = torch.zeros((3, 2, 5), dtype=torch.int64)
    assert position_strides(p, (0,)) == (10, 5, 1) and position_strides(p[:, :1], (0,)) == (10, 0, 1)
    assert position_strides(p[0], None) == (0, 5, 1) and position_strides(p[0], (0,)) == (5, 0, 1) and position_strides(p[0, 0], None) == (0, 0, 1)


def test_cpu_tensors_are_refused():
    table, n, one = torch.zeros((1, 2), dtype=torch.int32), _i32(1), _i32(2)
    pages, q = torch.zeros((4, 1, 16, 64), dtype=torch.bfloat16), torch.zeros((1, 1, 1, 64), dtype=torch.bfloat16)
    for call in (lambda: ktt.paged_reserve(table, n, n, one, one, 16, 1, _i32(0)), lambda: ktt.paged_release(table, n, n, one, one, 16, _i32(0)),
                 lambda: ktt.paged_bounds(pages, table, n), lambda: ktt.paged_select(q, pages[:, :, :2], table, n, 16, 2),
                 lambda: ktt.sdpa_paged(q, pages, pages, table[None], _i32(1)[None])):
        with pytest.raises((RuntimeError, ValueError), match="CUDA|no CPU"):
            call()
