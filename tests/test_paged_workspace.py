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


def _most(d, hk, capacity):
    """Dense rows of 1 GB or of one sequence, the offsets and the order of 512 sequences, and parts: two items of 128 rows for
    every SM of 148, d + 1 fp32 values a row."""
    return max(1 << 30, 4 * capacity * hk * d) + (64 + 3 * 512 + 2) * 4 + 256 + 2 * 148 * 128 * (d + 1) * 4


@pytest.mark.parametrize("bits", [16, 4])
def test_packed_calls_that_are_cut(built_lib, bits):
    """Launches that share the packed rows, and a buffer with more rows than its sequence: parts for a launch's rows alone."""
    for d, h, hk, batch, sq, capacity, total in ((128, 32, 8, 64, 128, 131072, 64 * 128), (128, 32, 8, 64, 128, 1 << 18, 64 * 128), (128, 8, 8, 1, 100, 8192, 65536),
                                                 (64, 8, 8, 1, 100, 8192, 65536)):
        need = _need(built_lib, bits, d, h, hk, batch, sq, capacity, total)
        dense = 4 * capacity * hk * d
        dense *= min(max((1 << 30) // dense, 1), batch)
        assert dense < need <= dense + _most(d, hk, capacity) - max(1 << 30, 4 * capacity * hk * d)
        assert need == _need(built_lib, bits, d, h, hk, batch, sq, capacity, 4 * total)


def test_no_call_needs_more(built_lib):
    g, cut = random.Random(1), 0
    for _ in range(3000):
        d, hk = g.choice([64, 128]), g.choice([1, 2, 8])
        h, batch, sq = hk * g.choice([1, 4, 7]), g.choice([1, 2, 3, 30, 700]), g.choice([65, 100, 129, 500, 3000])
        capacity = 16 << g.randrange(0, 14)
        total = g.choice([None, 1, 64, batch * sq // 2 + 1, batch * sq, 9 * batch * sq])
        need = _need(built_lib, g.choice([16, 4]), d, h, hk, batch, sq, capacity, total)
        assert need <= _most(d, hk, capacity), (d, h, hk, batch, sq, capacity, total)
        cut += need > 4 * capacity * hk * d * min(max((1 << 30) // (4 * capacity * hk * d), 1), batch, 512) + 16384
    assert cut > 100
