"""The pages of a paged cache that could matter most to a query: bounds of each page's keys, and the choice of pages by them.
(The reference attends to all keys of its static cache.)"""

import ctypes

import torch

from . import _lib, ops
from .paged import _offsets, _on_device, _pages, check_bounds, operator_offsets


def bounds_block(k_pages, block_table, lengths, bounds, what):
    """A ktt_b200_bounds_args block."""
    a = _lib.BoundsArgs()
    dim, batch, _ = _pages(a.cache, k_pages, k_pages, block_table, lengths, None, what)
    ops._require_cuda(bounds)
    check_bounds(bounds, k_pages, k_pages.shape[0], k_pages.shape[1], dim, what)
    a.batch, a.d, a.bounds = batch, dim, bounds.data_ptr()
    ops._set3(a.bounds_strides, bounds.stride()[:3])
    return a


def _bounds(k_pages, block_table, lengths, bounds, since):
    what = "paged_bounds"
    a = bounds_block(k_pages, block_table, lengths, bounds, what)
    ops._require_cuda(since)
    if since is not None:
        if since.dtype != torch.int32 or since.shape != lengths.shape or not since.is_contiguous() or since.device != lengths.device:
            raise ValueError("kohaku_tt_b200.paged_bounds: since must be a contiguous int32 [B]")
        a.since = since.data_ptr()
    with torch.cuda.device(k_pages.device):
        _lib.check(_lib.lib().ktt_b200_paged_bounds(ctypes.byref(a), ops._stream(k_pages.device)), what)


def _select(q, bounds, block_table, lengths, page_size, top, first, last, cu_seq_q):
    what = "paged_select"
    ops._require_cuda(q, bounds, block_table, lengths)
    packed = cu_seq_q is not None
    if q.dim() != (3 if packed else 4):
        raise ValueError("kohaku_tt_b200.paged_select: q must be [B, H, Sq, D], or packed [T, H, D] with cu_seq_q")
    if bounds.dim() != 4:
        raise ValueError("kohaku_tt_b200.paged_select: bounds must be bf16 [pages, Hk, 2, D]")
    pages, hk, _, dim = bounds.shape
    check_bounds(bounds, q, pages, hk, dim, what)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[1] < 1 or block_table.stride(1) != 1 or block_table.device != q.device:
        raise ValueError("kohaku_tt_b200.paged_select: block_table must be int32 [B, pages of a sequence] with dense rows")
    batch = block_table.shape[0]
    if lengths.dtype != torch.int32 or lengths.shape != (batch,) or not lengths.is_contiguous() or lengths.device != q.device:
        raise ValueError("kohaku_tt_b200.paged_select: lengths must be int32 [B]")
    if q.dtype != torch.bfloat16 or q.shape[-1] != dim or (not packed and q.shape[0] != batch):
        raise ValueError(f"kohaku_tt_b200.paged_select: q must be bf16, of {dim} columns and the table's sequences, got {q.dtype} {list(q.shape)}")
    rows = q.shape[0] if packed else q.shape[2]
    if rows >= 2 ** 31 or q.shape[1] > 65535 or hk > 4096:
        raise _lib.UnsupportedAttention("kohaku_tt_b200.paged_select: more rows or heads than the kernels count")
    if q.stride(-1) != 1 or q.data_ptr() % 16 or any(x % 8 for x in q.stride()[:-1]):
        q = q.clone(memory_format=torch.contiguous_format)
    a = _lib.SelectArgs()
    with torch.cuda.device(q.device):
        cu = None
        if packed:
            cu, _ = _offsets(cu_seq_q, batch, rows, q.device, what)
            a.cu_seqlens_q, a.total_q = cu.data_ptr(), rows
        a.batch, a.heads, a.kv_heads, a.sq, a.d = batch, q.shape[1], hk, 0 if packed else rows, dim
        a.page_size, a.table_width, a.pages, a.block_table, a.table_stride = ops.int32(page_size, "page_size", what), block_table.shape[1], pages, block_table.data_ptr(), block_table.stride(0)
        a.lengths, a.top, a.first, a.last = lengths.data_ptr(), *(ops.int32(x, name, what) for x, name in ((top, "top"), (first, "first"), (last, "last")))
        a.q, a.bounds = q.data_ptr(), bounds.data_ptr()
        ops._set3(a.q_strides, (ops._ths_strides if packed else ops._bhs_strides)(q))
        ops._set3(a.bounds_strides, bounds.stride()[:3])
        need = _lib.lib().ktt_b200_paged_select_workspace(ctypes.byref(a))
        if need < 0:
            _lib.check(_lib.ERR_UNSUPPORTED, what)
        tokens = rows if packed else batch * rows
        chosen, keys = lengths.new_empty((tokens, hk, a.top)), lengths.new_empty((tokens, hk))
        work = torch.empty((max(need, 16),), dtype=torch.uint8, device=q.device)
        a.chosen, a.keys, a.workspace, a.workspace_bytes = chosen.data_ptr(), keys.data_ptr(), work.data_ptr(), work.numel()
        _lib.check(_lib.lib().ktt_b200_paged_select(ctypes.byref(a), ops._stream(q.device)), what)
    return chosen, keys


@torch.library.custom_op("ktt_b200::_paged_bounds", mutates_args=("bounds",), device_types="cuda")
def _bounds_op(k_pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, bounds: torch.Tensor, since: torch.Tensor | None) -> None:
    _bounds(k_pages, block_table, lengths, bounds, since)


@_bounds_op.register_fake
def _(k_pages, block_table, lengths, bounds, since):
    return None


@torch.library.custom_op("ktt_b200::_paged_select", mutates_args=(), device_types="cuda")
def _select_op(q: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, page_size: int, top: int, first: int, last: int,
               cu_seq_q: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor]:
    return _select(q, bounds, block_table, lengths, page_size, top, first, last, cu_seq_q)


@_select_op.register_fake
def _(q, bounds, block_table, lengths, page_size, top, first, last, cu_seq_q):
    tokens = q.shape[0] if cu_seq_q is not None else q.shape[0] * q.shape[2]
    return lengths.new_empty((tokens, bounds.shape[1], top)), lengths.new_empty((tokens, bounds.shape[1]))


def paged_bounds(k_pages, block_table, lengths, bounds=None, since=None):
    """bounds, bf16 [pages, Hk, 2, D]: the least and the largest value of each channel over the keys of each page, as paged_read gives
    them, for the pages that hold the first lengths[b] keys of each sequence; a NaN among them stays one. Without bounds a new
    tensor, zero in all other pages; else it is written in place and returned. since (int32 [B] on the device): only the pages
    that keys since[b] .. lengths[b] - 1 lie in, of which the first keeps what its earlier keys left there. paged_append(bounds=)
    does that on the way. Bounds only ever widen, so those of a page that lost some of its keys (drafts that were not taken, a prompt cut
    back) have to be made again from the page's first key: by paged_release(bounds=), or here with since at that key. Pages in
    bf16 or 4 bits."""
    if bounds is None:
        dim = k_pages.shape[-1] if k_pages.dtype == torch.bfloat16 else k_pages.shape[-1] // 9 * 16
        bounds = k_pages.new_zeros((*k_pages.shape[:2], 2, dim), dtype=torch.bfloat16)
    eager = not torch.compiler.is_compiling() and _lib.native()
    if eager and eager.paged_bounds(k_pages, block_table, lengths, bounds, since):
        return bounds
    if ops.watched(k_pages, block_table, lengths, bounds):
        torch.ops.ktt_b200._paged_bounds(k_pages, block_table, lengths, bounds, since)
        return bounds
    _bounds(k_pages, block_table, lengths, bounds, since)
    return bounds


def paged_select(q, bounds, block_table, lengths, page_size, top, first=1, last=1, cu_seq_q=None):
    """The pages that each query token goes to, for each K / V head: (chosen, keys), which sdpa_paged takes for block_table and lengths.

    q: bf16 [B, H, Sq, D] (token b * Sq + s), or packed [T, H, D] with cu_seq_q (B + 1 offsets, a list, or int32 on the device).
    lengths int32 [B] count the keys with those of the call's own tokens, as in sdpa_paged: query i of n sees keys
    0 .. lengths[b] - n + i, and the pages that these lie in. Of them it goes to the `first` first ones, the `last` last ones (one at
    least: its own key is there), and those with the largest scores, `top` in all (or all, where there are no more). The score of a page is the
    largest logit that a key between its bounds (paged_bounds) could have with any query of the head's group,
        max over h of the sum over d of max(q[h, d] least[d], q[h, d] largest[d]),
    in 64 bits, which is exact where the products that are not 0 lie within a factor of 2^30 of one another (else each of the sum's additions
    rounds by 2^-53); ties go to the page that comes first. A score that is no number counts as infinite; an entry of
    block_table that names no page has score 0. (Where a least value is above the largest, as in a tensor that nothing was written to,
    it is not said which pages.)
    chosen int32 [tokens, Hk, top]: names of pages in the order of their places, -1 behind them. keys int32 [tokens, Hk]: the keys of
    those that the token sees (0: it sees none). Packed rows of no sequence see none. The two may share one allocation,
    which then lasts as long as either. H is a multiple of Hk, D 64 or 128. No gradients."""
    eager = not torch.compiler.is_compiling() and _lib.native()
    if eager and _on_device(cu_seq_q):
        out = eager.paged_select(q, bounds, block_table, lengths, page_size, top, first, last, cu_seq_q)
        if out is not None:
            return out
    if ops.watched(q, bounds, block_table, lengths):
        cu_seq_q = operator_offsets(cu_seq_q, block_table.shape[0], q.shape[0], q, "paged_select")
        return torch.ops.ktt_b200._paged_select(q, bounds, block_table, lengths, page_size, top, first, last, cu_seq_q)
    with torch.no_grad():
        return _select(q, bounds, block_table, lengths, int(page_size), int(top), int(first), int(last), cu_seq_q)
