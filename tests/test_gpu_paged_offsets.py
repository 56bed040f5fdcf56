"""Offsets of packed queries that lie outside of the rows there are: they are given on the device, where nobody checks them, so
they are taken as the nearest ones inside, whichever way a call takes. Operands lie between guard rows here."""

import ctypes

import pytest
import torch

from kohaku_tt_b200 import _lib
from tests.test_gpu_paged import _store, _x

pytestmark = pytest.mark.gpu

GUARD, FAR = 600, 2 ** 31 - 1
# what is given for T rows, and what it means (None: anything, inside)
OFFSETS = [
    (lambda t: [0, t, t + 330], lambda t: [0, t, t]),
    (lambda t: [-200, t // 2, t], lambda t: [0, t // 2, t]),
    (lambda t: [0, FAR, FAR], lambda t: [0, t, t]),
    (lambda t: [-FAR - 1, -5, t], lambda t: [0, 0, t]),
    (lambda t: [-FAR - 1, 3, FAR], lambda t: [0, 3, t]),
    (lambda t: [0, t - 1, t // 3], None),
    (lambda t: [t + 9, 2, -4], None),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("d,h,hk,t,sq,lengths", [
    (128, 2, 1, 200, 200, [3000, 1025]), (64, 2, 1, 200, 200, [3000, 1025]),     # cut along the keys
    (128, 8, 2, 200, 200, [300, 257]), (64, 8, 2, 200, 200, [300, 257]),
    (128, 8, 2, 200, 70, [300, 257]), (64, 2, 1, 200, 70, [3000, 1025]),        # more tokens than the call says a sequence has
    (128, 8, 2, 6, 6, [300, 257]), (64, 14, 2, 40, 40, [9000, 20])])
def test_offsets_outside(cuda, bits, d, h, hk, t, sq, lengths):
    page = 32
    wide = -(-max(lengths) // page)
    kp, vp = (_store(_x(2 * wide, hk, page, d, seed=i), bits, bool(i)).to(cuda) for i in range(2))
    table = torch.randperm(2 * wide, generator=torch.Generator().manual_seed(1)).to(device=cuda, dtype=torch.int32).view(2, wide)
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    q = _x(t + 2 * GUARD, h, d, seed=7).to(cuda)

    def attend(cu, causal):
        out = torch.full_like(q, 7.0)
        cu = torch.tensor(cu, dtype=torch.int32, device=cuda)
        a = _lib.PagedSdpaArgs()
        c = a.cache
        c.k, c.v, c.block_table, c.lengths = kp.data_ptr(), vp.data_ptr(), table.data_ptr(), lens.data_ptr()
        c.bits, c.page_size, c.kv_heads, c.table_width, c.pages, c.table_stride = bits, page, hk, wide, 2 * wide, wide
        for f in (c.k_strides, c.v_strides):
            f[0], f[1], f[2] = kp.stride()[:3]
        a.batch, a.heads, a.sq, a.d, a.total_q, a.causal, a.scale = 2, h, sq, d, t, causal, d ** -0.5
        a.q, a.out, a.cu_seqlens_q = q[GUARD:].data_ptr(), out[GUARD:].data_ptr(), cu.data_ptr()
        for f in (a.q_strides, a.out_strides):
            f[0], f[1], f[2] = 0, d, h * d
        need = _lib.lib().ktt_b200_paged_sdpa_workspace(ctypes.byref(a))
        work = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device=cuda)
        a.workspace, a.workspace_bytes = work.data_ptr(), need
        _lib.check(_lib.lib().ktt_b200_paged_sdpa(ctypes.byref(a), torch.cuda.current_stream().cuda_stream), "sdpa_paged")
        assert (out[:GUARD] == 7.0).all() and (out[GUARD + t:] == 7.0).all()
        assert (work[need:] == 0x5A).all()
        return out[GUARD:GUARD + t]

    for given, meant in OFFSETS:
        for causal in (0, 1):
            got = attend(given(t), causal)
            if meant:
                assert torch.equal(got, attend(meant(t), causal))
    torch.cuda.synchronize()
    _lib.device_status()
