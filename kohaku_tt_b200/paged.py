"""Keys and values cached in pages, in bf16 or 4 bits: appending rows with their rotation,
attention over the pages, and reading them back. (The reference's decode runs against a
static cache, `decode_step` here; pages let sequences share a pool, and 4 bits hold 3.5
times as many keys in it.)"""

import ctypes
import math
from collections.abc import Sequence

import torch

from . import _lib, attention, ops
from .rotary import check_positions, check_tables, dense_tables, fill_axes, pair_axes


def paged_cache(pages, kv_heads, page_size, dim, bits=16, device="cuda"):
    """(k_pages, v_pages), zero: bf16 [pages, kv_heads, page_size, dim], or with bits=4 uint8
    [pages, kv_heads, page_size, dim / 2 + dim / 16] (layout: ktt_b200_pages in include/ktt_b200.h).
    page_size is a multiple of 16, dim 64 or 128."""
    if bits not in (16, 4):
        raise ValueError(f"kohaku_tt_b200.paged_cache: bits must be 16 or 4, got {bits}")
    if dim not in (64, 128) or page_size < 16 or page_size % 16 or pages < 1 or kv_heads < 1:
        raise ValueError("kohaku_tt_b200.paged_cache: dim 64 or 128, a page size that is a multiple of 16, one page and head at least")
    shape = (pages, kv_heads, page_size, dim if bits == 16 else dim // 2 + dim // 16)
    dtype = torch.bfloat16 if bits == 16 else torch.uint8
    return torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)


def _pages(c, k_pages, v_pages, table, lengths, max_k, what):
    """Fills a ktt_b200_pages block; returns (head dim, batch, capacity)."""
    ops._require_cuda(k_pages, v_pages, table, lengths)
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        raise ValueError(f"kohaku_tt_b200.{what}: k_pages and v_pages must be [pages, Hk, page size, D] of one shape and type")
    if k_pages.dtype == torch.bfloat16:
        dim, bits = k_pages.shape[3], 16
    elif k_pages.dtype == torch.uint8 and k_pages.shape[3] % 9 == 0:
        dim, bits = k_pages.shape[3] // 9 * 16, 4
    else:
        raise _lib.UnsupportedAttention(f"kohaku_tt_b200.{what}: pages hold bf16, or uint8 rows of D / 2 + D / 16 bytes")
    for t in (k_pages, v_pages):
        if t.stride(3) != 1 or (bits == 4 and t.shape[2] > 1 and t.stride(2) != t.shape[3]):
            raise _lib.UnsupportedAttention(f"kohaku_tt_b200.{what}: a page's rows must be dense")
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[1] < 1 or table.stride(1) != 1:
        raise ValueError(f"kohaku_tt_b200.{what}: block_table must be int32 [B, pages of a sequence] with dense rows")
    if lengths.dtype != torch.int32 or lengths.shape != (table.shape[0],) or not lengths.is_contiguous():
        raise ValueError(f"kohaku_tt_b200.{what}: lengths must be int32 [B]")
    if any(t.device != k_pages.device for t in (v_pages, table, lengths)):
        raise ValueError(f"kohaku_tt_b200.{what}: pages, block_table and lengths must be on one device")
    cap = table.shape[1] * k_pages.shape[2]
    if max_k is not None:
        if max_k < 1:
            raise ValueError(f"kohaku_tt_b200.{what}: max_k must be 1 or more")
        cap = min(cap, int(max_k))
    c.k, c.v = k_pages.data_ptr(), v_pages.data_ptr()
    c.bits, c.page_size, c.kv_heads, c.table_width, c.pages = bits, k_pages.shape[2], k_pages.shape[1], table.shape[1], k_pages.shape[0]
    ops._set3(c.k_strides, k_pages.stride()[:3])
    ops._set3(c.v_strides, v_pages.stride()[:3])
    c.block_table, c.table_stride, c.lengths = table.data_ptr(), table.stride(0), lengths.data_ptr()
    c.max_keys = cap
    return dim, table.shape[0], cap


def _offsets(cu, batch, tokens, device, what):
    """(int32 [B + 1] on the device, longest or None) of offsets that are given on the host (checked here) or
    on the device (read by the kernels only)."""
    if isinstance(cu, torch.Tensor) and cu.is_cuda:
        if cu.dtype != torch.int32 or cu.shape != (batch + 1,) or not cu.is_contiguous() or cu.device != device:
            raise ValueError(f"kohaku_tt_b200.{what}: offsets must be int32 [{batch + 1}] on the operands' device")
        return cu, None
    host = attention.offsets(cu)
    if len(host) != batch + 1 or host[0] != 0 or host[-1] > tokens or any(x > y for x, y in zip(host, host[1:])):
        raise ValueError(f"kohaku_tt_b200.{what}: offsets must be [0, ..., at most {tokens}], {batch + 1} of them, and not decrease")
    return torch.tensor(host, dtype=torch.int32, device=device), max([0, *[y - x for x, y in zip(host, host[1:])]])


def _operand(t, name, heads, like, batch, rows, dim, packed, what):
    if rows >= 2 ** 31 or heads > 65535:
        raise _lib.UnsupportedAttention(f"kohaku_tt_b200.{what}: more rows or heads than the kernels count")
    shape = (rows, heads, dim) if packed else (batch, heads, rows, dim)
    if tuple(t.shape) != shape or t.dtype != torch.bfloat16 or t.device != like.device:
        raise ValueError(f"kohaku_tt_b200.{what}: {name} must be bf16 {list(shape)} on the pages' device, got {t.dtype} {list(t.shape)}")
    return ops._rows_contiguous(t)


def _on_device(cu):
    return cu is None or (isinstance(cu, torch.Tensor) and cu.is_cuda)


def operator_offsets(cu, batch, rows, like, what):
    """Offsets as an operator takes them, on the device."""
    return cu if _on_device(cu) else _offsets(cu, batch, rows, like.device, what)[0]


def check_bounds(bounds, like, pages, hk, dim, what):
    """The rules of a cache's bounds."""
    if tuple(bounds.shape) != (pages, hk, 2, dim) or bounds.dtype != torch.bfloat16 or bounds.device != like.device:
        raise ValueError(f"kohaku_tt_b200.{what}: bounds must be bf16 {[pages, hk, 2, dim]} on the pages' device, got {bounds.dtype} {list(bounds.shape)}")
    if bounds.stride(3) != 1:
        raise _lib.UnsupportedAttention(f"kohaku_tt_b200.{what}: the rows of bounds must be dense")


def _append(k, v, k_pages, v_pages, block_table, lengths, cos, sin, q, interleaved, cu_seq, lengths_out, positions=None, axes=None, bounds=None, granted=None):
    what = "paged_append"
    ops._require_cuda(k, v, q, cos, sin, lengths_out, positions, bounds, granted)
    at = _lib.AppendAtArgs()
    a = at.base
    dim, batch, cap = _pages(a.cache, k_pages, v_pages, block_table, lengths, None, what)
    packed = cu_seq is not None
    if k.dim() != (3 if packed else 4):
        raise ValueError("kohaku_tt_b200.paged_append: k must be [B, Hk, S, D], or packed [T, Hk, D] with cu_seq")
    rows, hk = k.shape[0] if packed else k.shape[2], k_pages.shape[1]
    k = _operand(k, "k", hk, k_pages, batch, rows, dim, packed, what)
    v = _operand(v, "v", hk, k_pages, batch, rows, dim, packed, what)
    strides = ops._ths_strides if packed else ops._bhs_strides
    with torch.cuda.device(k_pages.device):
        cu = None
        if packed:
            cu, _ = _offsets(cu_seq, batch, rows, k_pages.device, what)
            a.cu_seqlens = cu.data_ptr()
        if (cos is None) != (sin is None):
            raise ValueError("kohaku_tt_b200.paged_append: cos and sin go together")
        if cos is not None:
            a.pairs = check_tables(cos, sin, k_pages, dim, what)
            if positions is None and cos.shape[0] < cap:
                raise ValueError("kohaku_tt_b200.paged_append: the rotary tables must cover every cache position")
            cos, sin = dense_tables(cos, sin)
            a.cos, a.sin, a.table_stride, a.table_rows = cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.shape[0]
        if positions is None and axes is not None:
            raise ValueError("kohaku_tt_b200.paged_append: axes need positions")
        if positions is not None:
            if cos is None:
                raise ValueError("kohaku_tt_b200.paged_append: positions need rotary tables")
            axes = pair_axes(axes, cos.shape[1], what)
            check_positions(positions, axes, k, rows, what)
            fill_axes(at.positions, positions, axes)
        if bounds is not None:
            check_bounds(bounds, k_pages, k_pages.shape[0], hk, dim, what)
            at.bounds = bounds.data_ptr()
            ops._set3(at.bounds_strides, bounds.stride()[:3])
        q_out = None
        if q is not None:
            if q.dim() != k.dim() or q.shape[1] < 1:
                raise ValueError("kohaku_tt_b200.paged_append: q must be laid out like k, with its own heads")
            q = _operand(q, "q", q.shape[1], k_pages, batch, rows, dim, packed, what)
            q_out = ops._empty_like_rows(q)
            a.heads, a.q, a.q_out = q.shape[1], q.data_ptr(), q_out.data_ptr()
            ops._set3(a.q_strides, strides(q))
            ops._set3(a.q_out_strides, strides(q_out))
        if lengths_out is not None:
            if lengths_out.dtype != torch.int32 or lengths_out.shape != lengths.shape or not lengths_out.is_contiguous() or lengths_out.device != lengths.device:
                raise ValueError("kohaku_tt_b200.paged_append: lengths_out must be a contiguous int32 [B]")
            a.lengths_out = lengths_out.data_ptr()
        if granted is not None and (granted.dtype != torch.int32 or granted.shape != lengths.shape or not granted.is_contiguous() or granted.device != lengths.device):
            raise ValueError("kohaku_tt_b200.paged_append: granted must be a contiguous int32 [B]")
        a.batch, a.rows, a.d, a.interleaved = batch, rows, dim, int(interleaved)
        a.k, a.v = k.data_ptr(), v.data_ptr()
        ops._set3(a.k_strides, strides(k))
        ops._set3(a.v_strides, strides(v))
        if positions is not None or bounds is not None or granted is not None:
            given = None if granted is None else granted.data_ptr()
            _lib.check(_lib.lib().ktt_b200_paged_append_granted(ctypes.byref(at), given, ops._stream(k_pages.device)), what)
        else:
            _lib.check(_lib.lib().ktt_b200_paged_append(ctypes.byref(a), ops._stream(k_pages.device)), what)
    return q_out


def _read(k_pages, v_pages, block_table, lengths, max_k):
    a = _lib.ReadArgs()
    dim, batch, cap = _pages(a.cache, k_pages, v_pages, block_table, lengths, max_k, "paged_read")
    with torch.cuda.device(k_pages.device):
        k = torch.empty((batch, k_pages.shape[1], cap, dim), dtype=torch.bfloat16, device=k_pages.device)
        v = torch.empty_like(k)
        a.batch, a.rows, a.d = batch, cap, dim
        a.k_out, a.v_out = k.data_ptr(), v.data_ptr()
        ops._set3(a.k_strides, ops._bhs_strides(k))
        ops._set3(a.v_strides, ops._bhs_strides(v))
        _lib.check(_lib.lib().ktt_b200_paged_read(ctypes.byref(a), ops._stream(k_pages.device)), "paged_read")
    return k, v


def _attention_out(q, packed):
    """The output of sdpa_paged, by the queries that the caller gave (whose place in memory a graph does not know)."""
    return q.new_empty(q.shape) if packed else ops._out_like_query(ops._rows_contiguous(q), q.shape[-1])


def _sdpa(q, k_pages, v_pages, block_table, lengths, causal, scale, cu_seq_q, max_q, max_k):
    what = "sdpa_paged"
    ops._require_cuda(q)
    a = _lib.PagedSdpaArgs()
    dim, batch, _ = _pages(a.cache, k_pages, v_pages, block_table, lengths, max_k, what)
    packed = cu_seq_q is not None
    if q.dim() != (3 if packed else 4):
        raise ValueError("kohaku_tt_b200.sdpa_paged: q must be [B, H, Sq, D], or packed [T, H, D] with cu_seq_q")
    rows = q.shape[0] if packed else q.shape[2]
    q = _operand(q, "q", q.shape[1], k_pages, batch, rows, dim, packed, what)
    out = _attention_out(q, packed)
    if q.data_ptr() % 16 or any(x % 8 for x in q.stride()[:-1]):
        q = q.clone(memory_format=torch.contiguous_format)   # (rows that the kernels cannot read in place)
    strides = ops._ths_strides if packed else ops._bhs_strides
    with torch.cuda.device(q.device):
        cu = None
        if packed:
            cu, longest = _offsets(cu_seq_q, batch, rows, q.device, what)
            a.cu_seqlens_q, a.total_q = cu.data_ptr(), rows
            max_q = longest if max_q is None and longest is not None else rows if max_q is None else int(max_q)
            if max_q < 0 or (longest is not None and max_q < longest):
                raise ValueError("kohaku_tt_b200.sdpa_paged: max_q is less than the longest sequence")
            max_q = min(max_q, rows)
        a.batch, a.heads, a.sq, a.d = batch, q.shape[1], max_q if packed else rows, dim
        a.causal, a.scale = int(causal), float(scale) if scale is not None else 1.0 / math.sqrt(dim)
        a.q, a.out = q.data_ptr(), out.data_ptr()
        ops._set3(a.q_strides, strides(q))
        ops._set3(a.out_strides, strides(out))
        need = _lib.lib().ktt_b200_paged_sdpa_workspace(ctypes.byref(a))
        if need < 0:
            _lib.check(_lib.ERR_UNSUPPORTED, what)
        work = torch.empty((max(need, 16),), dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = work.data_ptr(), work.numel()
        _lib.check(_lib.lib().ktt_b200_paged_sdpa(ctypes.byref(a), ops._stream(q.device)), what)
    return out


def _chosen(q, k_pages, v_pages, chosen, keys, scale, max_k):
    """sdpa_paged with a table of each token's and K / V head's own."""
    what = "sdpa_paged"
    ops._require_cuda(q, chosen, keys)
    if chosen.dim() != 3 or chosen.dtype != torch.int32 or chosen.shape[2] < 1 or chosen.shape[1] != k_pages.shape[1]:
        raise ValueError("kohaku_tt_b200.sdpa_paged: block_table of three dimensions must be int32 [tokens, Hk, pages]")
    if keys.dtype != torch.int32 or keys.shape != chosen.shape[:2]:
        raise ValueError("kohaku_tt_b200.sdpa_paged: lengths must be int32 [tokens, Hk] there")
    if q.dim() not in (3, 4):
        raise ValueError("kohaku_tt_b200.sdpa_paged: q must be [B, H, Sq, D] or [T, H, D]")
    packed = q.dim() == 3
    batch, rows = (1, q.shape[0]) if packed else (q.shape[0], q.shape[2])
    if batch * rows != chosen.shape[0]:
        raise ValueError(f"kohaku_tt_b200.sdpa_paged: tables of {chosen.shape[0]} tokens for {batch * rows}")
    chosen, keys = chosen.contiguous(), keys.contiguous()
    a = _lib.PagedSdpaArgs()
    dim, _, _ = _pages(a.cache, k_pages, v_pages, chosen.view(-1, chosen.shape[2]), keys.view(-1), max_k, what)
    q = _operand(q, "q", q.shape[1], k_pages, batch, rows, dim, packed, what)
    out = _attention_out(q, packed)
    if q.data_ptr() % 16 or any(x % 8 for x in q.stride()[:-1]):
        q = q.clone(memory_format=torch.contiguous_format)
    strides = ops._ths_strides if packed else ops._bhs_strides
    with torch.cuda.device(q.device):
        a.batch, a.heads, a.sq, a.d = batch, q.shape[1], rows, dim
        a.scale = float(scale) if scale is not None else 1.0 / math.sqrt(dim)
        a.q, a.out = q.data_ptr(), out.data_ptr()
        ops._set3(a.q_strides, strides(q))
        ops._set3(a.out_strides, strides(out))
        need = _lib.lib().ktt_b200_paged_sdpa_chosen_workspace(ctypes.byref(a))
        if need < 0:
            _lib.check(_lib.ERR_UNSUPPORTED, what)
        work = torch.empty((max(need, 16),), dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = work.data_ptr(), work.numel()
        _lib.check(_lib.lib().ktt_b200_paged_sdpa_chosen(ctypes.byref(a), ops._stream(q.device)), what)
    return out


# ---- operators for compiled graphs (which pass tensors, not lists) ---------------------------

@torch.library.custom_op("ktt_b200::_paged_append", mutates_args=("k_pages", "v_pages", "lengths_out"), device_types="cuda")
def _append_op(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
               cos: torch.Tensor | None, sin: torch.Tensor | None, q: torch.Tensor | None, interleaved: bool, cu_seq: torch.Tensor | None,
               lengths_out: torch.Tensor | None) -> torch.Tensor:
    out = _append(k, v, k_pages, v_pages, block_table, lengths, cos, sin, q, interleaved, cu_seq, lengths_out)
    return k.new_empty((0,)) if out is None else out


@torch.library.custom_op("ktt_b200::_paged_append_at", mutates_args=("k_pages", "v_pages", "lengths_out", "bounds"), device_types="cuda")
def _append_at_op(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
                  cos: torch.Tensor | None, sin: torch.Tensor | None, q: torch.Tensor | None, interleaved: bool, cu_seq: torch.Tensor | None,
                  lengths_out: torch.Tensor | None, positions: torch.Tensor | None, axes: Sequence[int] | None, bounds: torch.Tensor | None,
                  granted: torch.Tensor | None) -> torch.Tensor:
    """With positions, bounds or granted. (As arguments of the operator above that are None by default they would be lost on their way.)"""
    out = _append(k, v, k_pages, v_pages, block_table, lengths, cos, sin, q, interleaved, cu_seq, lengths_out, positions, axes, bounds, granted)
    return k.new_empty((0,)) if out is None else out


@_append_op.register_fake
def _(k, v, k_pages, v_pages, block_table, lengths, cos, sin, q, interleaved, cu_seq, lengths_out):
    return k.new_empty((0,)) if q is None else ops._empty_like_rows(q)


@_append_at_op.register_fake
def _(k, v, k_pages, v_pages, block_table, lengths, cos, sin, q, interleaved, cu_seq, lengths_out, positions, axes, bounds, granted):
    return k.new_empty((0,)) if q is None else ops._empty_like_rows(q)


@torch.library.custom_op("ktt_b200::_paged_read", mutates_args=(), device_types="cuda")
def _read_op(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, max_k: int | None) -> tuple[torch.Tensor, torch.Tensor]:
    return _read(k_pages, v_pages, block_table, lengths, max_k)


@_read_op.register_fake
def _(k_pages, v_pages, block_table, lengths, max_k):
    dim = k_pages.shape[3] if k_pages.dtype == torch.bfloat16 else k_pages.shape[3] // 9 * 16
    cap = block_table.shape[1] * k_pages.shape[2]
    shape = (block_table.shape[0], k_pages.shape[1], cap if max_k is None else min(cap, max_k), dim)
    return k_pages.new_empty(shape, dtype=torch.bfloat16), k_pages.new_empty(shape, dtype=torch.bfloat16)


@torch.library.custom_op("ktt_b200::_sdpa_paged", mutates_args=(), device_types="cuda")
def _sdpa_op(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, causal: bool,
             scale: float | None, cu_seq_q: torch.Tensor | None, max_q: int | None, max_k: int | None) -> torch.Tensor:
    return _sdpa(q, k_pages, v_pages, block_table, lengths, causal, scale, cu_seq_q, max_q, max_k)


@_sdpa_op.register_fake
def _(q, k_pages, v_pages, block_table, lengths, causal, scale, cu_seq_q, max_q, max_k):
    return _attention_out(q, cu_seq_q is not None)


@torch.library.custom_op("ktt_b200::_sdpa_paged_chosen", mutates_args=(), device_types="cuda")
def _chosen_op(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, chosen: torch.Tensor, keys: torch.Tensor, scale: float | None,
               max_k: int | None) -> torch.Tensor:
    return _chosen(q, k_pages, v_pages, chosen, keys, scale, max_k)


@_chosen_op.register_fake
def _(q, k_pages, v_pages, chosen, keys, scale, max_k):
    return _attention_out(q, q.dim() == 3)


# ---- the entry points ------------------------------------------------------------------------

def paged_append(k, v, k_pages, v_pages, block_table, lengths, cos=None, sin=None, q=None, interleaved=False,
                 cu_seq=None, lengths_out=None, positions=None, axes=None, bounds=None, granted=None):
    """Writes new keys and values behind what sequences have in a paged cache, the keys rotated on the way
    (and the step's queries alongside), in one launch.

    k, v: bf16 [B, Hk, S, D], or packed [T, Hk, D] with cu_seq (B + 1 offsets, a list, or int32 on the
    device; rows that no sequence covers are not read). No two sequences may append to one page in one call. Row i of sequence b goes to place lengths[b] + i:
    row p % page_size of page block_table[b, p // page_size]. An entry that is no page of the cache (-1, say)
    takes nothing, nor does a place past the table. lengths: int32 [B] on the device, keys cached so far; they
    are not changed, lengths_out (optional, another buffer) receives the new ones.
    cos, sin: rotary_table's, one row per place of the cache; without them keys go in as they are. Rotation as
    in `rotary` (interleaved; columns past 2 * pairs are copied), the result in bf16.
    q: bf16 [B, H, S, D] or [T, H, D]; returned rotated (None without q; packed rows of no sequence undefined).
    positions, axes: as in `rotary`, where rows turn by positions other than their places (pictures in a
    prompt; packed rows: [T], or [axes, T]); the tables then need not cover the places.
    bounds: a cache's bounds (paged_bounds), which are kept up to date for the pages that the new keys go to;
    what those held before, and nothing else, must be in the bounds already (a sequence that was cut back inside a page: paged_release).
    granted: paged_reserve's, int32 [B] on the device: only the first granted[b] new rows of each sequence go into pages and bounds and
    count in lengths_out (queries are rotated all the same). Without it all rows do, also those that the reservation had no room for: what of
    them fits goes into the last page that the sequence has, and lengths_out counts the others too.
    Pages of 4 bits (paged_cache(bits=4)) hold each 64 channels of a row as codes 0 to 15 of
    least + step * code, step = bf16((most - least) / 15): codes are the nearest. No gradients."""
    interleaved = bool(interleaved)
    # Eager calls on plain CUDA tensors are served by C++ in one step.
    eager = not torch.compiler.is_compiling() and _lib.native()
    if eager and _on_device(cu_seq):
        out = eager.paged_append(k, v, k_pages, v_pages, block_table, lengths, cos, sin, q, interleaved, cu_seq, lengths_out, positions, axes, bounds, granted)
        if out is not NotImplemented:
            return out
    if ops.watched(k, v, k_pages, v_pages, block_table, lengths, q):
        cu_seq = operator_offsets(cu_seq, block_table.shape[0], k.shape[0], k_pages, "paged_append")
        if positions is None and axes is None and bounds is None and granted is None:
            out = torch.ops.ktt_b200._paged_append(k, v, k_pages, v_pages, block_table, lengths, cos, sin, q, interleaved, cu_seq, lengths_out)
        else:
            out = torch.ops.ktt_b200._paged_append_at(k, v, k_pages, v_pages, block_table, lengths, cos, sin, q, interleaved, cu_seq, lengths_out,
                                                      positions, axes, bounds, granted)
        return out if q is not None else None
    with torch.no_grad():
        return _append(k, v, k_pages, v_pages, block_table, lengths, cos, sin, q, interleaved, cu_seq, lengths_out, positions, axes, bounds, granted)


def paged_read(k_pages, v_pages, block_table, lengths, max_k=None):
    """(k, v), bf16 [B, Hk, capacity, D]: the first lengths[b] keys and values of each sequence out of its
    pages, as their values where the pages hold 4 bits; zeros behind them and where there is no page.
    capacity: block_table's, or max_k where that is less."""
    eager = not torch.compiler.is_compiling() and _lib.native()
    if eager:
        out = eager.paged_read(k_pages, v_pages, block_table, lengths, max_k)
        if out is not None:
            return out
    if ops.watched(k_pages, v_pages, block_table, lengths):
        return torch.ops.ktt_b200._paged_read(k_pages, v_pages, block_table, lengths, max_k)
    with torch.no_grad():
        return _read(k_pages, v_pages, block_table, lengths, max_k)


def sdpa_paged(q, k_pages, v_pages, block_table, lengths, is_causal=True, scale=None, cu_seq_q=None, max_q=None,
               max_k=None):
    """Attention of q [B, H, Sq, D] over the first lengths[b] keys of each sequence's pages; Sq may be one
    token, a few, or a chunk of a prompt. Packed: q [T, H, D] with cu_seq_q (B + 1 offsets, a list, or int32 on
    the device, then best with max_q, no less than the longest sequence, and taken inside of the T rows); rows that no
    sequence covers are left undefined.

    Pages as in paged_append, bf16 or 4 bits, D 64 or 128, H a multiple of Hk. lengths (int32 [B] on the
    device) count the keys with those of the call's own tokens, which are appended first. Under is_causal the
    diagonal is aligned to the end: query i of n sees keys 0 .. lengths[b] - n + i. A row that sees no key
    gets zeros. max_k: no sequence has more keys (default: what block_table has room for; longer ones are
    cut); an entry of block_table within a length that is no page of the cache reads as zeros. A key that some of a sequence's queries see and others do not must be finite. Weights are
    rounded to bf16 for their product with the values, to fp16 in chunks of prompts over 4-bit pages. No gradients.

    block_table [tokens, Hk, pages] with lengths [tokens, Hk] (paged_select's): each query token has its own pages
    for each K / V head, and sees the first lengths[t, h] keys of them; q [B, H, Sq, D] (token b * Sq + s) or
    [T, H, D], without offsets."""
    causal = bool(is_causal)
    eager = not torch.compiler.is_compiling() and _lib.native()
    if block_table.dim() == 3:
        if cu_seq_q is not None or max_q is not None:
            raise ValueError("kohaku_tt_b200.sdpa_paged: with a table for each token there are no offsets")
        if eager:
            out = eager.sdpa_paged_chosen(q, k_pages, v_pages, block_table, lengths, scale, max_k)
            if out is not None:
                return out
        if ops.watched(q, k_pages, v_pages, block_table, lengths):
            return torch.ops.ktt_b200._sdpa_paged_chosen(q, k_pages, v_pages, block_table, lengths, scale, max_k)
        with torch.no_grad():
            return _chosen(q, k_pages, v_pages, block_table, lengths, scale, max_k)
    if eager and _on_device(cu_seq_q):
        out = eager.sdpa_paged(q, k_pages, v_pages, block_table, lengths, causal, scale, cu_seq_q, max_q, max_k)
        if out is not None:
            return out
    if ops.watched(q, k_pages, v_pages, block_table, lengths):
        if not _on_device(cu_seq_q):
            cu_seq_q, longest = _offsets(cu_seq_q, block_table.shape[0], q.shape[0], q.device, "sdpa_paged")
            if max_q is not None and max_q < longest:
                raise ValueError("kohaku_tt_b200.sdpa_paged: max_q is less than the longest sequence")
            max_q = longest if max_q is None else max_q
        return torch.ops.ktt_b200._sdpa_paged(q, k_pages, v_pages, block_table, lengths, causal, scale, cu_seq_q, max_q, max_k)
    with torch.no_grad():
        return _sdpa(q, k_pages, v_pages, block_table, lengths, causal, scale, cu_seq_q, max_q, max_k)
