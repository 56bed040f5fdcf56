"""The C entry with queries at any 4 bytes and outputs at any 8, which it takes: chunks then run on the general kernel where the
tensor kernels cannot address them. Against float64."""

import ctypes

import pytest
import torch

from kohaku_tt_b200 import _lib
from oracle import paged_oracle as po
from tests.test_gpu_paged import _cache, _near, _x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("d,h,hk,n,lengths", [(128, 8, 2, 4, [300, 0, 65]), (64, 4, 2, 1, [300, 0, 65]), (128, 4, 2, 130, [300, 0, 65]), (64, 2, 1, 130, [2500, 0, 129])])
@pytest.mark.parametrize("q_off,out_off", [(2, 0), (0, 4), (6, 12), (8, 8)])
def test_operands_at_odd_places(cuda, bits, packed, d, h, hk, n, lengths, q_off, out_off):
    b, page = len(lengths), 16
    kp, vp, table = _cache(bits, d, hk, page, lengths)
    qs = _x(b, h, n, d, seed=7)
    want, mags, sizes = po.attend([q.double() for q in qs], kp.nan_to_num(0.0) if bits == 16 else kp, vp.nan_to_num(0.0) if bits == 16 else vp, table, lengths, True, d ** -0.5)
    rows = torch.zeros(b * n * h * d + 64, dtype=torch.bfloat16, device=cuda)
    flat = (qs.transpose(1, 2) if packed else qs).reshape(-1)
    rows[q_off:q_off + flat.numel()] = flat.to(cuda)
    out = torch.full_like(rows, 7.0)
    kp, vp, table = kp.to(cuda), vp.to(cuda), table.to(cuda)
    lens, cu = torch.tensor(lengths, dtype=torch.int32, device=cuda), torch.arange(b + 1, dtype=torch.int32, device=cuda) * n
    a = _lib.PagedSdpaArgs()
    c = a.cache
    c.k, c.v, c.block_table, c.lengths = kp.data_ptr(), vp.data_ptr(), table.data_ptr(), lens.data_ptr()
    c.bits, c.page_size, c.kv_heads, c.table_width, c.pages, c.table_stride = bits, page, hk, table.shape[1], kp.shape[0], table.shape[1]
    for f, t in ((c.k_strides, kp), (c.v_strides, vp)):
        f[0], f[1], f[2] = t.stride()[:3]
    a.batch, a.heads, a.sq, a.d, a.causal, a.scale = b, h, n, d, 1, d ** -0.5
    a.q, a.out = rows.data_ptr() + 2 * q_off, out.data_ptr() + 2 * out_off
    for f in (a.q_strides, a.out_strides):
        f[0], f[1], f[2] = (0, d, h * d) if packed else (h * n * d, n * d, d)
    if packed:
        a.cu_seqlens_q, a.total_q = cu.data_ptr(), b * n
    need = _lib.lib().ktt_b200_paged_sdpa_workspace(ctypes.byref(a))
    work = torch.empty(need, dtype=torch.uint8, device=cuda)
    a.workspace, a.workspace_bytes = work.data_ptr(), need
    _lib.check(_lib.lib().ktt_b200_paged_sdpa(ctypes.byref(a), torch.cuda.current_stream().cuda_stream), "sdpa_paged")
    got = out[out_off:out_off + flat.numel()].view((b, n, h, d) if packed else (b, h, n, d))
    assert (out[:out_off] == 7.0).all() and (out[out_off + flat.numel():] == 7.0).all()
    _near(list(got.transpose(1, 2) if packed else got), want, mags, sizes, bits == 4)
