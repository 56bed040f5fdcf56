"""Block tables of a paged cache, kept on the device: pages for the tokens that requests bring, out of a list of free
ones, with each token's position and slot; and pages given back. (The reference has a static cache and no tables.)"""

import ctypes

import torch

from . import _lib, ops
from .selection import bounds_block


def _tables(block_table, lengths, free, count, page_size, count_out, what):
    """A ktt_b200_tables block."""
    ops._require_cuda(block_table, lengths, free, count, count_out)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[1] < 1 or block_table.stride(1) != 1:
        raise ValueError(f"kohaku_tt_b200.{what}: block_table must be int32 [B, pages of a sequence] with dense rows")
    batch = block_table.shape[0]
    for name, t, shape in (("lengths", lengths, (batch,)), ("count", count, (1,)), ("count_out", count_out, (1,)), ("free", free, (free.numel(),))):
        if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != block_table.device:
            raise ValueError(f"kohaku_tt_b200.{what}: {name} must be a contiguous int32 {list(shape)} on the table's device")
    a = _lib.Tables()
    a.batch, a.table_width, a.page_size = batch, block_table.shape[1], ops.int32(page_size, "page_size", what)
    a.block_table, a.table_stride, a.lengths = block_table.data_ptr(), block_table.stride(0), lengths.data_ptr()
    a.free_pages, a.pool, a.count, a.count_out = free.data_ptr(), free.numel(), count.data_ptr(), count_out.data_ptr()
    return a


def _vector(t, name, like, what):
    ops._require_cuda(t)
    if t.dtype != torch.int32 or t.shape != like.shape or not t.is_contiguous() or t.device != like.device:
        raise ValueError(f"kohaku_tt_b200.{what}: {name} must be a contiguous int32 [B] on the table's device")


def _reserve(block_table, lengths, added, free, count, page_size, tokens, count_out):
    what = "paged_reserve"
    a = _tables(block_table, lengths, free, count, page_size, count_out, what)
    _vector(added, "added", lengths, what)
    if tokens < 0:
        raise ValueError("kohaku_tt_b200.paged_reserve: tokens must be 0 or more")
    with torch.cuda.device(block_table.device):
        cu = lengths.new_empty((lengths.shape[0] + 1,))
        positions, slots, granted = lengths.new_empty((tokens,)), lengths.new_empty((tokens,), dtype=torch.int64), torch.empty_like(lengths)
        _lib.check(_lib.lib().ktt_b200_paged_reserve(ctypes.byref(a), added.data_ptr(), tokens, cu.data_ptr(), positions.data_ptr(), slots.data_ptr(),
                                                     granted.data_ptr(), ops._stream(block_table.device)), what)
    return cu, positions, slots, granted


def _release(block_table, lengths, kept, free, count, page_size, count_out, k_pages, bounds):
    what = "paged_release"
    a = _tables(block_table, lengths, free, count, page_size, count_out, what)
    _vector(kept, "kept", lengths, what)
    if (k_pages is None) != (bounds is None):
        raise ValueError("kohaku_tt_b200.paged_release: k_pages and bounds go together")
    edges = None
    if bounds is not None:
        edges = bounds_block(k_pages, block_table, lengths, bounds, what)
        if k_pages.shape[2] != page_size:
            raise ValueError(f"kohaku_tt_b200.paged_release: pages of {k_pages.shape[2]} keys, and page_size {page_size}")
    with torch.cuda.device(block_table.device):
        _lib.check(_lib.lib().ktt_b200_paged_release_bounds(ctypes.byref(a), kept.data_ptr(), None if edges is None else ctypes.byref(edges),
                                                            ops._stream(block_table.device)), what)


@torch.library.custom_op("ktt_b200::_paged_reserve", mutates_args=("block_table", "count_out"), device_types="cuda")
def _reserve_op(block_table: torch.Tensor, lengths: torch.Tensor, added: torch.Tensor, free: torch.Tensor, count: torch.Tensor, page_size: int, tokens: int,
                count_out: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return _reserve(block_table, lengths, added, free, count, page_size, tokens, count_out)


@_reserve_op.register_fake
def _(block_table, lengths, added, free, count, page_size, tokens, count_out):
    batch = lengths.shape[0]
    return lengths.new_empty((batch + 1,)), lengths.new_empty((tokens,)), lengths.new_empty((tokens,), dtype=torch.int64), lengths.new_empty((batch,))


@torch.library.custom_op("ktt_b200::_paged_release", mutates_args=("block_table", "free", "count_out", "bounds"), device_types="cuda")
def _release_op(block_table: torch.Tensor, lengths: torch.Tensor, kept: torch.Tensor, free: torch.Tensor, count: torch.Tensor, page_size: int,
                count_out: torch.Tensor, k_pages: torch.Tensor | None, bounds: torch.Tensor | None) -> None:
    _release(block_table, lengths, kept, free, count, page_size, count_out, k_pages, bounds)


@_release_op.register_fake
def _(block_table, lengths, kept, free, count, page_size, count_out, k_pages, bounds):
    return None


def paged_reserve(block_table, lengths, added, free, count, page_size, tokens, count_out):
    """Pages for added[b] new tokens of each sequence (int32 [B] on the device) behind the lengths[b] keys that it has, in one launch
    and without a trip to the host: (cu_seq, positions, slots, granted).

    block_table int32 [B, W] is written in place: entries ceil(lengths / page_size) .. of each row that the new tokens reach. free
    int32 [pool], with a place for each of the pool's pages 0 .. pool - 1, count int32 [1]: free[:count] are those that no sequence
    has. They are taken from the end, sequence by sequence; neither is changed, count_out (int32 [1], another buffer) receives how
    many are left. lengths are not changed either.
    granted int32 [B]: added[b], or 0 for the first sequence that the list, or its row of the table, has no room for and for all
    behind it; their new entries become -1, and they can be asked for again later. Given to paged_append, it keeps their rows out of the
    cache and out of lengths_out; where no call can run short it may be left out. What selections and attention give for their queries
    is of no use.
    The new tokens are packed, row i of sequence b at cu_seq[b] + i, as paged_append and sdpa_paged take them: cu_seq int32 [B + 1];
    for `tokens` rows (the sum of added; 0: not wanted), positions int32, lengths[b] + i, and slots int64, page * page_size + row in the
    page, which is where the token's row lies in a buffer [pages * page_size, ...]; -1 in rows behind the last sequence's, and
    in the slots of sequences that were granted nothing. The four may share one allocation, which then lasts as long as any of them (clone what is
    kept for long, or saved). At most 4096 sequences."""
    eager = not torch.compiler.is_compiling() and _lib.native()
    if eager:
        out = eager.paged_reserve(block_table, lengths, added, free, count, page_size, tokens, count_out)
        if out is not None:
            return out
    if ops.watched(block_table, lengths, added, free, count):
        return torch.ops.ktt_b200._paged_reserve(block_table, lengths, added, free, count, page_size, tokens, count_out)
    return _reserve(block_table, lengths, added, free, count, int(page_size), int(tokens), count_out)


def paged_release(block_table, lengths, kept, free, count, page_size, count_out, k_pages=None, bounds=None):
    """Cuts sequences back to their first kept[b] keys (int32 [B] on the device; 0: the sequence has ended; lengths[b]: it goes on):
    the pages that hold none of those go to free[count:], sequence by sequence, and their entries of block_table become -1;
    count_out (int32 [1], another buffer than count) receives the new number. lengths are not changed: they are kept's from then on.
    Entries that name no page give nothing back. A page that two sequences share must not be given back by both,
    nor cut, with bounds, by the one that has fewer keys in it.
    k_pages, bounds: those of a cache with bounds (paged_bounds), which are made again, in a launch beside it, for the pages that
    sequences are cut in: of the keys that are left there, so that later appends and selections know nothing of the others."""
    eager = not torch.compiler.is_compiling() and _lib.native()
    if eager and eager.paged_release(block_table, lengths, kept, free, count, page_size, count_out, k_pages, bounds):
        return
    if ops.watched(block_table, lengths, kept, free, count):
        torch.ops.ktt_b200._paged_release(block_table, lengths, kept, free, count, page_size, count_out, k_pages, bounds)
        return
    _release(block_table, lengths, kept, free, count, int(page_size), count_out, k_pages, bounds)
