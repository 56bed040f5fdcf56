"""What the entries of a server's steps refuse where they are not plain, without a GPU (no kernel is launched in this file)."""

import ctypes

import pytest
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
    a.block_table = a.lengths = a.count = 4096
    a.free_pages, a.count_out = 1 << 20, 8192
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


def test_fake_tensors_reach_the_fake_operators():
    """Under FakeTensorMode nothing reads a pointer: each entry gives what its operator says of shapes and types, traced or not."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    import kohaku_tt_b200 as ktt

    b, h, hk, d, page, wide, pool, t, top = 3, 8, 2, 64, 16, 20, 50, 9, 4

    def step(q, k, v, kp, vp, bounds, table, lengths, added, free, count, left, after, cos, sin):
        cu, at, slots, granted = ktt.paged_reserve(table, lengths, added, free, count, page, t, left)
        turned = ktt.paged_append(k, v, kp, vp, table, lengths, cos, sin, q=q, cu_seq=cu, lengths_out=after, positions=at.expand(3, t), axes=tuple(i % 3 for i in range(d // 2)),
                                  bounds=bounds, granted=granted)
        plain = ktt.paged_append(k, v, kp, vp, table, lengths, q=q, cu_seq=[0, 4, 4, 9])
        assert ktt.paged_append(k, v, kp, vp, table, lengths, cu_seq=[0, 4, 4, 9]) is None
        chosen, keys = ktt.paged_select(turned, bounds, table, after, page, top, cu_seq_q=cu)
        other, _ = ktt.paged_select(turned, bounds, table, after, page, top, cu_seq_q=[0, 4, 4, 9])
        out = ktt.sdpa_paged(turned, kp, vp, chosen, keys)
        every = ktt.sdpa_paged(turned, kp, vp, table, after, cu_seq_q=[0, 4, 4, 9])
        again = ktt.paged_bounds(kp, table, after)
        dense = ktt.paged_read(kp, vp, table, after, max_k=100)
        ktt.paged_release(table, after, lengths, free, left, page, count, k_pages=kp, bounds=bounds)
        r = ktt.rotary(q, k, cos, sin, positions=at)
        s = ktt.rotary(q, None, cos, sin, positions=at.expand(3, t), axes=tuple(i % 3 for i in range(d // 2)))
        return cu, at, slots, granted, turned, plain, chosen, keys, other, out, every, again, *dense, *r, s[0]

    def bf16(*shape):
        return torch.empty(shape, dtype=torch.bfloat16, device="cuda")

    def i32(*shape):
        return torch.empty(shape, dtype=torch.int32, device="cuda")

    with FakeTensorMode() as mode:
        args = (bf16(t, h, d), bf16(t, hk, d), bf16(t, hk, d), bf16(pool, hk, page, d), bf16(pool, hk, page, d), bf16(pool, hk, 2, d), i32(b, wide), i32(b), i32(b), i32(pool), i32(1), i32(1),
                i32(b), torch.empty((wide * page, d // 2), device="cuda"), torch.empty((wide * page, d // 2), device="cuda"))
        got = step(*args)
    want = [((b + 1,), torch.int32), ((t,), torch.int32), ((t,), torch.int64), ((b,), torch.int32), ((t, h, d), torch.bfloat16), ((t, h, d), torch.bfloat16), ((t, hk, top), torch.int32),
            ((t, hk), torch.int32), ((t, hk, top), torch.int32), ((t, h, d), torch.bfloat16), ((t, h, d), torch.bfloat16), ((pool, hk, 2, d), torch.bfloat16), ((b, hk, 100, d), torch.bfloat16),
            ((b, hk, 100, d), torch.bfloat16), ((t, h, d), torch.bfloat16), ((t, hk, d), torch.bfloat16), ((t, h, d), torch.bfloat16)]
    assert [(tuple(x.shape), x.dtype) for x in got] == want and all(x.device.type == "cuda" for x in got)
    # Outside of the mode too, as the tensors themselves are fake; and a traced graph has every operator.
    chosen, keys = ktt.paged_select(got[4], args[5], args[6], args[12], page, top, cu_seq_q=got[0])
    assert chosen.fake_mode is mode and tuple(chosen.shape) == (t, hk, top)
    with mode:
        graph = make_fx(step)(*args)
    names = {str(n.target) for n in graph.graph.nodes if n.op == "call_function"}
    for name in ("_paged_reserve", "_paged_append_at", "_paged_append", "_paged_select", "_sdpa_paged_chosen", "_sdpa_paged", "_paged_bounds", "_paged_read", "_paged_release", "_rotary",
                 "_rotary_axes"):
        assert f"ktt_b200.{name}.default" in names, (name, names)


def test_written_bounds_that_lie_on_one_another(built_lib):
    """Strides against each other, not each alone; layouts whose rows are apart pass (they are refused for a batch of none, behind this check)."""
    def status(strides, pages=4, kv_heads=2, d=64):
        b = _bounds(strides=strides, pages=pages, kv_heads=kv_heads, d=d)
        b.batch = 70000
        first = built_lib.ktt_b200_paged_bounds(ctypes.byref(b), None)
        assert first == _lib.ERR_UNSUPPORTED and "65535" in _lib.last_error()
        x = _append(batch=70000, d=d)      # (the number of sequences is checked after the bounds there)
        x.bounds, x.base.cache.pages, x.base.cache.kv_heads = 4096, pages, kv_heads
        for i, s in enumerate(strides):
            x.bounds_strides[i] = s
        assert built_lib.ktt_b200_paged_append_at(ctypes.byref(x), None) == _lib.ERR_UNSUPPORTED
        return "on one another" in _lib.last_error()

    for strides in ((64, 64, 64), (128, 64, 64), (64, 128, 64), (192, 128, 64), (256, 64, 64), (256, 128, 120), (64, 256, 128), (0, 128, 64), (256, 128, 0), (-128, 128, 64),
                    (128, 256, -128), (2 ** 62, 2 ** 62, 64)):
        assert status(strides), strides
    for strides in ((256, 128, 64), (64, 512, 256), (128, 512, 64), (256, 64, 128), (-256, 128, -64), (4096, 64, 1024), (2 ** 62, 128, 64), (2 ** 62, 2 ** 61, 64)):
        assert not status(strides), strides
    assert not status((0, 128, 64), pages=1) and not status((128, 0, 64), kv_heads=1) and status((128, 0, 64), kv_heads=2) and status((100, 128, 64), pages=2)


def test_whole_numbers_of_an_argument_block():
    from kohaku_tt_b200 import ops

    assert [ops.int32(x, "x", "test") for x in (0, -(2 ** 31), 2 ** 31 - 1, 16.0)] == [0, -(2 ** 31), 2 ** 31 - 1, 16]
    for x in (2 ** 31, -(2 ** 31) - 1, 2 ** 32 + 16):
        with pytest.raises(_lib.UnsupportedAttention, match="must fit 32 bits"):
            ops.int32(x, "x", "test")


def test_more_pages_and_heads_than_blocks(built_lib):
    """Grids past 2^31 blocks are refused before anything is launched (past 2^32 their lower bits were)."""
    b = _bounds(page_size=16, table_width=1 << 26, kv_heads=256, table_stride=1 << 26, pages=1)
    b.bounds_strides[1] = 128
    assert built_lib.ktt_b200_paged_bounds(ctypes.byref(b), None) == _lib.ERR_UNSUPPORTED and "2^34" in _lib.last_error()
    x = _append(rows=1 << 30, cu_seqlens=4096)
    x.bounds, x.base.cache.kv_heads = 4096, 4096
    for i, s in enumerate((4096 * 128, 128, 64)):
        x.bounds_strides[i] = s
    assert built_lib.ktt_b200_paged_append_granted(ctypes.byref(x), None, None) == _lib.ERR_UNSUPPORTED and "2^34" in _lib.last_error()


def test_outputs_of_tables_over_their_inputs(built_lib):
    """What some blocks of a launch read while others write is refused, in whole or in part; beside one another is fine (refused for their stride, behind it)."""
    base = dict(block_table=1 << 20, lengths=4096, free_pages=8192, count=12288, count_out=16384)      # 2 sequences, a list of 8

    def reserve(cu=None, positions=None, slots=None, granted=None, **kw):
        status = built_lib.ktt_b200_paged_reserve(ctypes.byref(_tables(**{**base, **kw})), 20480, 3, cu, positions, slots, granted, None)
        return status == _lib.ERR_BAD_ARGUMENT and "overlap" in _lib.last_error()

    for given in (4096, 4100, 20480, 20484, 8192, 8192 + 28, 12288):      # lengths, added, the list, the count
        assert reserve(granted=given) and reserve(cu=given) and reserve(positions=given) and reserve(slots=given & ~7), given
        if given != 12288:
            assert reserve(count_out=given)
    assert reserve(cu=4096 - 8) and reserve(slots=4096 - 16) and reserve(positions=20480 - 8)

    def release(kept=20480, **kw):
        status = built_lib.ktt_b200_paged_release(ctypes.byref(_tables(**{**base, **kw})), kept, None)
        return status == _lib.ERR_BAD_ARGUMENT and "overlap" in _lib.last_error()

    for given in (4096, 4100, 20480, 20484, 8192, 8192 + 28):
        assert release(count_out=given), given
    assert release(kept=8192) and release(kept=8192 + 28) and release(lengths=8188) and release(count=8200)
