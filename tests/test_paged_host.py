"""The paged cache and rotary entries without a GPU: the layout of 4-bit pages, and what the C entries refuse
(no kernel is launched in this file)."""

import ctypes

import pytest
import torch

import kohaku_tt_b200 as ktt
from kohaku_tt_b200 import _lib, paged
from oracle import paged_oracle as po


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [False, True])
def test_every_nibble_of_a_block_is_used_once(dim, value):
    assert sorted(po.places(dim, value).tolist()) == list(range(16 * dim))
    x = torch.randn((3, 2, 32, dim), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    pages = po.pack(x, value)
    assert pages.shape == (3, 2, 32, dim // 2 + dim // 16)
    code, step, least = po.quantise(x)
    assert torch.equal(po.values(pages, value), po.worth(code, step, least))
    # The nearest of 16 evenly spaced values (of a step rounded to bf16, 2^-9 of it: 15 x that at the far end).
    off = (po.worth(code, step, least) - x.float()).abs().unflatten(-1, (-1, 64))
    assert (off <= step.unsqueeze(-1) * (0.5 + 15 * 2.0 ** -8)).all()


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


BAD_PAGES = [(dict(bits=8), "16 or 4 bits"), (dict(page_size=24), "multiple of 16"), (dict(page_size=0), "multiple of 16"), (dict(kv_heads=0), "positive"),
             (dict(pages=0), "positive"), (dict(table_width=0), "positive"), (dict(k=4104), "16-byte aligned"), (dict(table_width=1 << 28, page_size=64), "2^30")]


@pytest.mark.parametrize("kw,text", BAD_PAGES)
def test_pages_that_no_entry_takes(built_lib, kw, text):
    append, read, sdpa = _lib.AppendArgs(cache=_pages(**kw)), _lib.ReadArgs(cache=_pages(**kw)), _lib.PagedSdpaArgs(cache=_pages(**kw))
    for a, entry in ((append, built_lib.ktt_b200_paged_append), (read, built_lib.ktt_b200_paged_read), (sdpa, built_lib.ktt_b200_paged_sdpa)):
        a.d = 128
        a.batch = 1
        assert entry(ctypes.byref(a), None) == _lib.ERR_UNSUPPORTED
        assert text in _lib.last_error()


def test_odd_strides_and_dims_are_refused(built_lib):
    a = _lib.ReadArgs(cache=_pages())
    a.batch = a.rows = 1
    a.d = 96
    assert built_lib.ktt_b200_paged_read(ctypes.byref(a), None) == _lib.ERR_UNSUPPORTED
    a.d = 128
    a.cache.k_strides[0] = 4097
    assert built_lib.ktt_b200_paged_read(ctypes.byref(a), None) == _lib.ERR_UNSUPPORTED
    a.cache.k_strides[0] = 4096
    assert built_lib.ktt_b200_paged_read(ctypes.byref(a), None) == _lib.ERR_BAD_ARGUMENT   # no outputs
    a.k_out = a.v_out = 4100
    assert built_lib.ktt_b200_paged_read(ctypes.byref(a), None) == _lib.ERR_UNSUPPORTED    # not aligned


def test_append_refusals(built_lib):
    def args(**kw):
        a = _lib.AppendArgs(cache=_pages())
        a.batch, a.rows, a.d, a.k, a.v = 1, 1, 128, 4096, 4096
        for name, x in kw.items():
            setattr(a, name, x)
        return a

    for kw in (dict(batch=0), dict(rows=-1), dict(k=None), dict(heads=2), dict(cos=4096), dict(cos=4096, sin=4096, pairs=65, table_rows=4),
               dict(cos=4096, sin=4096, pairs=4, table_rows=0), dict(lengths_out=4096), dict(batch=4, lengths_out=4096 + 12), dict(batch=4, lengths_out=4096 - 12)):
        assert built_lib.ktt_b200_paged_append(ctypes.byref(args(**kw)), None) == _lib.ERR_BAD_ARGUMENT, kw
    assert built_lib.ktt_b200_paged_append(ctypes.byref(args(rows=0)), None) == 0      # nothing to do
    assert built_lib.ktt_b200_paged_append(None, None) == _lib.ERR_BAD_ARGUMENT


def test_attention_refusals(built_lib):
    def args(**kw):
        a = _lib.PagedSdpaArgs(cache=_pages())
        a.batch, a.heads, a.sq, a.d, a.scale, a.q, a.out = 1, 4, 1, 128, 0.1, 4096, 4096
        for name, x in kw.items():
            setattr(a, name, x)
        return a

    for kw, rc in ((dict(heads=3), _lib.ERR_UNSUPPORTED), (dict(scale=0.0), _lib.ERR_UNSUPPORTED), (dict(scale=float("nan")), _lib.ERR_UNSUPPORTED),
                   (dict(batch=0), _lib.ERR_BAD_ARGUMENT), (dict(q=None), _lib.ERR_BAD_ARGUMENT), (dict(sq=-1), _lib.ERR_BAD_ARGUMENT)):
        assert built_lib.ktt_b200_paged_sdpa(ctypes.byref(args(**kw)), None) == rc, kw
    assert built_lib.ktt_b200_paged_sdpa(ctypes.byref(args(sq=0)), None) == 0


def test_a_diagonal_at_the_key_lengths_end_is_the_forward_s_alone(built_lib):
    """causal 3 needs key lengths; packed calls with key lengths take it or none; the backward takes neither."""
    def args(**kw):
        a = _lib.AttnArgs()
        a.batch, a.heads, a.kv_heads, a.sq, a.sk, a.d, a.dv, a.scale = 1, 1, 1, 8, 8, 64, 64, 0.1
        a.q = a.k = a.v = a.out = a.key_lengths = 4096
        for name, x in kw.items():
            setattr(a, name, x)
        return ctypes.byref(a)

    packed = dict(cu_seqlens_q=4096, cu_seqlens_k=4096, total_q=8, total_k=8)
    assert built_lib.ktt_b200_sdpa_supported(args(causal=3)) and built_lib.ktt_b200_sdpa_supported(args(causal=3, **packed))
    for kw in (dict(causal=3, key_lengths=None), dict(causal=2, **packed), dict(causal=4), dict(causal=-1)):
        assert not built_lib.ktt_b200_sdpa_supported(args(**kw)), kw
        assert built_lib.ktt_b200_sdpa_forward(args(**kw), None) == _lib.ERR_UNSUPPORTED, kw
    for kw in (dict(causal=3), dict(causal=3, **packed), dict(causal=0, **packed)):
        assert not built_lib.ktt_b200_sdpa_backward_supported(args(**kw)), kw
        assert built_lib.ktt_b200_sdpa_backward(args(**kw), None) == _lib.ERR_UNSUPPORTED, kw


def test_rotary_refusals(built_lib):
    def args(**kw):
        a = _lib.RotaryArgs()
        a.batch, a.rows, a.heads, a.d, a.pairs, a.dtype, a.table_rows = 1, 1, 1, 64, 32, _lib.MASK_BF16, 4
        a.q = a.q_out = a.cos = a.sin = 4096
        for name, x in kw.items():
            setattr(a, name, x)
        return a

    for kw, rc in ((dict(pairs=33), _lib.ERR_BAD_ARGUMENT), (dict(pairs=0), _lib.ERR_BAD_ARGUMENT), (dict(heads=0), _lib.ERR_BAD_ARGUMENT),
                   (dict(dtype=1), _lib.ERR_UNSUPPORTED), (dict(d=1026, pairs=1), _lib.ERR_UNSUPPORTED), (dict(kv_heads=1), _lib.ERR_BAD_ARGUMENT),
                   (dict(cos=None), _lib.ERR_BAD_ARGUMENT), (dict(table_rows=0), _lib.ERR_BAD_ARGUMENT)):
        assert built_lib.ktt_b200_rotary(ctypes.byref(args(**kw)), None) == rc, kw
    assert built_lib.ktt_b200_rotary(ctypes.byref(args(rows=0)), None) == 0
    f = (ctypes.c_double * 2)(1.0, 0.1)
    assert built_lib.ktt_b200_rotary_table(4096, 4096, 0, 2, f, 1.0, None) == _lib.ERR_BAD_ARGUMENT
    assert built_lib.ktt_b200_rotary_table(4096, 4096, 4, 257, f, 1.0, None) == _lib.ERR_BAD_ARGUMENT
    assert built_lib.ktt_b200_rotary_table(None, 4096, 4, 2, f, 1.0, None) == _lib.ERR_BAD_ARGUMENT


def test_host_tensors_and_offsets_are_refused(built_lib):
    k, v = ktt.paged_cache(3, 2, 16, 64, device="cpu")
    table, lengths = torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ktt.sdpa_paged(torch.zeros((1, 2, 1, 64), dtype=torch.bfloat16), k, v, table, lengths)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ktt.paged_read(k, v, table, lengths)
    for cu in ([0], [1, 2, 3], [0, 3, 2], [0, 2, 9]):
        with pytest.raises(ValueError, match="offsets"):
            paged._offsets(cu, 2, 8, torch.device("cpu"), "paged_append")
    for kw in (dict(bits=8), dict(dim=96), dict(page_size=20), dict(pages=0)):
        with pytest.raises(ValueError):
            ktt.paged_cache(**{**dict(pages=1, kv_heads=1, page_size=16, dim=64, device="cpu"), **kw})


def test_struct_sizes(built_lib):
    # Natural alignment on both sides: offsets that would shift on a mismatch.
    assert _lib.Pages.pages.offset == 32 and ctypes.sizeof(_lib.Pages) == 120
    assert _lib.AppendArgs.batch.offset == 120 and _lib.RotaryArgs.q.offset == 40 and _lib.PagedSdpaArgs.total_q.offset == 136
