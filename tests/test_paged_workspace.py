"""The workspace of attention over pages, from the sizes of a call alone (no kernel is launched in this file)."""

import ctypes
import random

import pytest

from kohaku_tt_b200 import _lib


def _need(lib, bits, d, h, hk, batch, sq, capacity, total_q=None):
    a = _lib.PagedSdpaArgs()
    c = a.cache
    c.k = c.v = c.block_table = c.lengths = 4096
    c.bits, c.page_size, c.kv_heads, c.table_width, c.pages, c.table_stride = bits, 16, hk, capacity // 16, 9, capacity // 16
    for f in (c.k_strides, c.v_strides):
        f[0], f[1], f[2] = 16 * hk * d, 16 * d, d
    a.batch, a.heads, a.sq, a.d, a.scale, a.q, a.out = batch, h, sq, d, 0.1, 4096, 4096
    if total_q is not None:
        a.cu_seqlens_q, a.total_q = 4096, total_q
    need = lib.ktt_b200_paged_sdpa_workspace(ctypes.byref(a))
    assert need > 0, _lib.last_error()
    return need


def _dense(d, hk, batch, capacity):
    """Bytes of dense rows: of as many sequences as take 1 GB, or of one; and how many those are."""
    one = 4 * capacity * hk * d
    count = min(max((1 << 30) // one, 1), batch, 512)
    return count * one, count


def _more(bits, d, h, hk, count, capacity, rows):
    """What comes to them: the offsets and the order of 512 sequences; over 4 bits the powers of two of each 64 keys, and a copy of the
    queries with theirs; parts: two items of 128 rows for every SM of 148, d + 1 fp32 values a row."""
    four = hk * count * -(-capacity // 128) * 2 * 4 + rows * h * (2 * d + 4) + 3 * 256
    return (64 + 3 * 512 + 2) * 4 + 256 + (four if bits == 4 else 0) + 2 * 148 * 128 * (d + 1) * 4


@pytest.mark.parametrize("bits", [16, 4])
def test_packed_calls_that_are_cut(built_lib, bits):
    """Launches that share the packed rows, and a buffer with more rows than its sequence: parts for a launch's rows alone."""
    for d, h, hk, batch, sq, capacity, total in ((128, 32, 8, 64, 128, 131072, 64 * 128), (128, 32, 8, 64, 128, 1 << 18, 64 * 128), (128, 8, 8, 1, 100, 8192, 65536),
                                                 (64, 8, 8, 1, 100, 8192, 65536)):
        need = _need(built_lib, bits, d, h, hk, batch, sq, capacity, total)
        dense, count = _dense(d, hk, batch, capacity)
        assert dense < need <= dense + _more(bits, d, h, hk, count, capacity, total)
        copies = 3 * total * h * (2 * d + 4) if bits == 4 else 0     # (more rows behind the sequences)
        assert abs(_need(built_lib, bits, d, h, hk, batch, sq, capacity, 4 * total) - need - copies) < 1024


def test_no_call_needs_more(built_lib):
    g, cut = random.Random(1), 0
    for _ in range(3000):
        d, hk = g.choice([64, 128]), g.choice([1, 2, 8])
        h, batch, sq = hk * g.choice([1, 4, 7]), g.choice([1, 2, 3, 30, 700]), g.choice([65, 100, 129, 500, 3000])
        capacity = 16 << g.randrange(0, 14)
        total = g.choice([None, 1, 64, batch * sq // 2 + 1, batch * sq, 9 * batch * sq])
        bits = g.choice([16, 4])
        need = _need(built_lib, bits, d, h, hk, batch, sq, capacity, total)
        dense, count = _dense(d, hk, batch, capacity)
        parts = 2 * 148 * 128 * (d + 1) * 4
        most = dense + _more(bits, d, h, hk, count, capacity, batch * sq if total is None else total)
        assert need <= most, (d, h, hk, batch, sq, capacity, total)
        cut += need > most - parts
    assert cut > 100
