"""Rotary positions: tables of cosines and sines, scaled for long contexts or not, and the
rotation of queries and keys with its gradient. (The reference's ktt.rotary,
csrc/aten/nn/aten_fused.cpp:30-43, turns whole heads in the half layout; decode_step has
that in its one launch.)"""

import ctypes

import torch

from . import _lib, ops

_DTYPES = {torch.bfloat16: _lib.MASK_BF16, torch.float16: _lib.MASK_F16, torch.float32: _lib.MASK_F32}
SCALINGS = (None, "linear", "base", "parts")


def rotary_frequencies(dim, base=10000.0, scaling=None, factor=1.0, original=None, fast=32.0, slow=1.0):
    """(frequencies, scale): the angle per position of each of dim / 2 pairs as Python floats, and
    what the cosines and sines are multiplied by. See rotary_table."""
    f, m = (ctypes.c_double * 256)(), ctypes.c_double()
    _lib.check(_lib.lib().ktt_b200_rotary_frequencies(f, ctypes.byref(m), int(dim), base, _scaling(scaling), factor,
                                                      0.0 if original is None else original, fast, slow), "rotary_table")
    return f[:dim // 2], m.value


def _scaling(name):
    if name not in SCALINGS:
        raise ValueError(f"kohaku_tt_b200.rotary_table: scaling must be one of {SCALINGS}, got {name!r}")
    return SCALINGS.index(name)


def rotary_table(positions, dim, base=10000.0, scaling=None, factor=1.0, original=None, fast=32.0, slow=1.0,
                 device="cuda"):
    """(cos, sin), fp32 [positions, dim / 2]: those of the angles p f_i, f_i = base^(-2 i / dim), of
    positions p = 0, 1, ... Angles are taken in 64 bits, so far positions keep their precision.

    scaling, for contexts `factor` times as long as a model was trained for:
      "linear"  f_i / factor: positions are interpolated;
      "base"    base times factor^(dim / (dim - 2)): the slowest pair is interpolated, the fastest kept;
      "parts"   pairs that turn `fast` times or more within the `original` context keep their
                frequency, those that turn `slow` times or less get f_i / factor; one that turns r times
                between them keeps (r - slow) / (fast - slow) of it and has f_i / factor for the rest
                (a ramp in the turns, not in i); cos and sin are multiplied by 0.1 ln(factor) + 1."""
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError("kohaku_tt_b200: rotary tables are made on CUDA devices only; there is no CPU fallback")
    scaling, original = _scaling(scaling), 0.0 if original is None else original
    eager = not torch.compiler.is_compiling() and _lib.native()
    if eager:
        index = torch.cuda.current_device() if device.index is None else device.index
        out = eager.rotary_table(positions, dim, base, scaling, factor, original, fast, slow, index)
        if out is not None:
            return out
    return torch.ops.ktt_b200._rotary_table(int(positions), int(dim), base, scaling, factor, original, fast, slow, device)


@torch.library.custom_op("ktt_b200::_rotary_table", mutates_args=(), device_types="cuda")
def _table_op(positions: int, dim: int, base: float, scaling: int, factor: float, original: float, fast: float, slow: float,
              device: torch.device) -> tuple[torch.Tensor, torch.Tensor]:
    """The tables as an operator, for compiled graphs and for modes that watch operators."""
    f, scale = rotary_frequencies(dim, base, SCALINGS[scaling], factor, original, fast, slow)
    if positions < 1:
        raise ValueError("kohaku_tt_b200.rotary_table: one position at least")
    pairs = len(f)
    with torch.cuda.device(device):
        cos = torch.empty((positions, pairs), dtype=torch.float32, device=device)
        sin = torch.empty_like(cos)
        host = (ctypes.c_double * pairs)(*f)
        _lib.check(_lib.lib().ktt_b200_rotary_table(cos.data_ptr(), sin.data_ptr(), positions, pairs, host, scale,
                                                    ops._stream(cos.device)), "rotary_table")
    return cos, sin


@_table_op.register_fake
def _(positions, dim, base, scaling, factor, original, fast, slow, device):
    shape = (positions, dim // 2)
    return torch.empty(shape, dtype=torch.float32, device=device), torch.empty(shape, dtype=torch.float32, device=device)


def check_tables(cos, sin, like, dim, what):
    """The rules of cos / sin for operands of `dim` columns; returns the pairs that turn."""
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.dim() != 2 or cos.shape != sin.shape:
        raise ValueError(f"kohaku_tt_b200.{what}: cos and sin must be fp32 [positions, pairs] of one shape")
    if cos.device != like.device or sin.device != like.device:
        raise ValueError(f"kohaku_tt_b200.{what}: cos and sin must be on the operands' device")
    if cos.requires_grad or sin.requires_grad:
        raise ValueError(f"kohaku_tt_b200.{what}: the tables get no gradient")
    if cos.shape[0] < 1 or cos.shape[1] < 1 or 2 * cos.shape[1] > dim:
        raise ValueError(f"kohaku_tt_b200.{what}: 1 to {dim // 2} pairs turn, got tables {tuple(cos.shape)}")
    return cos.shape[1]


def dense_tables(cos, sin):
    if cos.stride(1) != 1 or sin.stride(1) != 1 or cos.stride(0) != sin.stride(0):
        return cos.contiguous(), sin.contiguous()
    return cos, sin


def _check(q, k, cos, sin, positions):
    what = "rotary"
    for x in (q, k):
        if x is None:
            continue
        if x.dim() not in (3, 4) or x.dim() != q.dim():
            raise ValueError("kohaku_tt_b200.rotary: q and k must be [B, H, S, D] or packed [T, H, D]")
        if x.dtype not in _DTYPES or x.dtype != q.dtype or x.device != q.device:
            raise _lib.UnsupportedAttention("kohaku_tt_b200.rotary: q and k must be bf16, fp16 or fp32, of one type and device")
        same = x.shape[-1] == q.shape[-1] and (x.shape[0] == q.shape[0] if x.dim() == 3 else x.shape[0] == q.shape[0] and x.shape[2] == q.shape[2])
        if not same:
            raise ValueError("kohaku_tt_b200.rotary: q and k differ in more than their heads")
    if max(q.shape[:-1]) >= 2 ** 31 or q.shape[1] > 65535 or (k is not None and k.shape[1] > 65535):
        raise _lib.UnsupportedAttention("kohaku_tt_b200.rotary: more rows or heads than the kernel counts")
    check_tables(cos, sin, q, q.shape[-1], what)
    rows = q.shape[0] if q.dim() == 3 else q.shape[2]
    if positions is None:
        if cos.shape[0] < rows:
            raise ValueError(f"kohaku_tt_b200.rotary: tables of {cos.shape[0]} positions for {rows} rows")
        return
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device:
        raise ValueError("kohaku_tt_b200.rotary: positions must be an int32 or int64 tensor on the operands' device")
    fits = positions.shape == (rows,) or (q.dim() == 4 and positions.shape in ((q.shape[0], rows), (1, rows)))
    if not fits:
        raise ValueError(f"kohaku_tt_b200.rotary: one position per row ([{rows}], or [batch, {rows}]), got {tuple(positions.shape)}")


def _run(q, k, cos, sin, positions, interleaved, inverse):
    """The launch, after the checks: (q', k' or None)."""
    ops._require_cuda(q, k, cos, sin, positions)
    q = ops._rows_contiguous(q)
    k = None if k is None else ops._rows_contiguous(k)
    cos, sin = dense_tables(cos, sin)
    strides = ops._ths_strides if q.dim() == 3 else ops._bhs_strides
    with torch.cuda.device(q.device):
        q_out, k_out = ops._empty_like_rows(q), None if k is None else ops._empty_like_rows(k)
        if q.numel() == 0 and (k is None or k.numel() == 0):
            return q_out, k_out
        a = _lib.RotaryArgs()
        a.batch, a.rows = (1, q.shape[0]) if q.dim() == 3 else (q.shape[0], q.shape[2])
        a.heads, a.kv_heads, a.d = q.shape[1], 0 if k is None else k.shape[1], q.shape[-1]
        a.pairs, a.interleaved, a.inverse, a.dtype = cos.shape[1], int(interleaved), int(inverse), _DTYPES[q.dtype]
        a.q, a.q_out = q.data_ptr(), q_out.data_ptr()
        ops._set3(a.q_strides, strides(q))
        ops._set3(a.q_out_strides, strides(q_out))
        if k is not None:
            a.k, a.k_out = k.data_ptr(), k_out.data_ptr()
            ops._set3(a.k_strides, strides(k))
            ops._set3(a.k_out_strides, strides(k_out))
        a.cos, a.sin, a.table_stride, a.table_rows = cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.shape[0]
        if positions is not None:
            a.positions, a.positions_are_64 = positions.data_ptr(), int(positions.dtype == torch.int64)
            a.position_strides[0] = positions.stride(0) if positions.dim() == 2 and positions.shape[0] > 1 else 0
            a.position_strides[1] = positions.stride(-1)
        _lib.check(_lib.lib().ktt_b200_rotary(ctypes.byref(a), ops._stream(q.device)), "rotary")
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """The rotation; its gradient is the inverse rotation, by the same node (so it can be
    differentiated again)."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, interleaved, inverse):
        ctx.save_for_backward(cos, sin, positions)
        ctx.how = (interleaved, inverse)
        ctx.set_materialize_grads(False)
        return _run(q, k, cos, sin, positions, interleaved, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        cos, sin, positions = ctx.saved_tensors
        interleaved, inverse = ctx.how
        rest = (cos, sin, positions, interleaved, not inverse)
        if dq is None and dk is None:
            return (None,) * 7
        if dq is None:
            return (None, _Rotary.apply(dk, None, *rest)[0], None, None, None, None, None)
        dq, dk = _Rotary.apply(dq, dk, *rest)
        return dq, dk, None, None, None, None, None


@torch.library.custom_op("ktt_b200::_rotary", mutates_args=(), device_types="cuda")
def _rotary_op(q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None,
               interleaved: bool, inverse: bool) -> list[torch.Tensor]:
    """The rotation as an operator, for compiled graphs."""
    q_out, k_out = _run(q, k, cos, sin, positions, interleaved, inverse)
    return [q_out] if k_out is None else [q_out, k_out]


@_rotary_op.register_fake
def _(q, k, cos, sin, positions, interleaved, inverse):
    return [ops._empty_like_rows(x) for x in (q, k) if x is not None]


def _setup(ctx, inputs, output):
    _, k, cos, sin, positions, interleaved, inverse = inputs
    ctx.save_for_backward(cos, sin, positions)
    ctx.how = (interleaved, inverse, [x.shape for x in output])


def _op_backward(ctx, grads):
    cos, sin, positions = ctx.saved_tensors
    interleaved, inverse, shapes = ctx.how
    some = next((g for g in grads if g is not None), None)
    if some is None:
        return (None,) * 7
    grads = [some.new_zeros(shape) if g is None else g for g, shape in zip(grads, shapes)]
    got = torch.ops.ktt_b200._rotary(grads[0], grads[1] if len(grads) > 1 else None, cos, sin, positions, interleaved, not inverse)
    return got[0], got[1] if len(got) > 1 else None, None, None, None, None, None


_rotary_op.register_autograd(_op_backward, setup_context=_setup)


def rotary(q, k, cos, sin, positions=None, interleaved=False):
    """Rotary positions of q [B, H, S, D] and k [B, Hk, S, D] (packed: [T, H, D] and [T, Hk, D]; k may be
    None): (q', k'), new tensors laid out like q and k, with gradients.

    cos, sin: fp32 [P, R / 2], R <= D even (rotary_table). Columns past R are copied. The others turn in
    pairs: (i, i + R / 2), or neighbours (2 i, 2 i + 1) with interleaved=True, by
        y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin
    in fp32, products and sum rounded one by one, the result once to q's type (bf16, fp16 or fp32).
    positions: int32 or int64 on the device, [S] or [B, S] (packed [T]), read by the kernel and clamped to
    the tables' rows; without them row s has position s."""
    interleaved = bool(interleaved)
    # Eager calls on plain CUDA tensors are served by C++ in one step (None: not such a call).
    eager = not torch.compiler.is_compiling() and _lib.native()
    if eager:
        out = eager.rotary(q, k, cos, sin, positions, interleaved)
        if out is not None:
            return out
    _check(q, k, cos, sin, positions)
    if torch.compiler.is_compiling():
        out = torch.ops.ktt_b200._rotary(q, k, cos, sin, positions, interleaved, False)
        return (out[0], None if k is None else out[1])
    return _Rotary.apply(q, k, cos, sin, positions, interleaved, False)
