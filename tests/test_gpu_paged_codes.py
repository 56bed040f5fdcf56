"""Codes of groups whose steps are subnormal: a step of a few of the least bf16 values is rounded by as much as half of one, and
the farthest values then lie past 15 of them; and what codes are worth where the least value is far below the step."""

import pytest
import torch

import kohaku_tt_b200 as ktt
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu

LEAST = 2.0 ** -133     # of the bf16 values above 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("least", [0.0, -7 * LEAST, -100 * LEAST])
def test_ranges_of_a_few_of_the_least_values(cuda, d, least):
    """Ranges of 1 to 255 of them: codes, steps and least values to the bit, 0 to 15 of them."""
    n = 256
    part = torch.rand((n, 1, d), generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    part[..., 0::64], part[..., 1::64] = 0.0, 1.0
    whole = torch.arange(n, dtype=torch.float64)[:, None, None]
    x = (least + torch.round(part * whole) * LEAST).to(torch.bfloat16)
    kp, vp = ktt.paged_cache(n // 16, 1, 16, d, bits=4, device=cuda)
    table = torch.arange(n // 16, dtype=torch.int32, device=cuda)[None]
    xd = x.transpose(0, 1)[None].to(cuda)
    ktt.paged_append(xd, xd, kp, vp, table, torch.zeros(1, dtype=torch.int32, device=cuda))
    want = po.quantise(x)
    assert (want[0].max() == 15) and (want[1] > 0).any()
    for pages, value in ((kp, False), (vp, True)):
        got = po.unpack(pages.cpu(), value)
        for a, b in zip(got, want):
            assert torch.equal(a.transpose(1, 2).reshape(b.shape), b)


@pytest.mark.parametrize("d", [64, 128])
def test_a_code_s_worth_is_rounded_once(cuda, d):
    """least + step * code of all 16 codes, least values of 2^-12 to 2^-40 of the step on both sides: against the sum in 64 bits, rounded to the
    nearest bf16, ties to even."""
    n = 256
    x = torch.zeros((n, 1, d), dtype=torch.bfloat16)
    steps = 1 + torch.arange(n) % 128 / 128.0
    for g in range(0, d, 64):
        for c in range(64):
            x[:, 0, g + c] = ((c % 16) * steps).to(torch.bfloat16)
    pages = {value: po.pack(x.view(n // 16, 16, 1, d).transpose(1, 2), value) for value in (False, True)}
    least = (2.0 ** -(12 + torch.arange(n) % 29).double() * (1 - 2 * (torch.arange(n) // 29 % 2))).to(torch.bfloat16)
    for pool in pages.values():     # the least values themselves, beside the codes
        words = pool.view(n // 16, 1, 1, 16 * (d // 2 + d // 16))[..., 8 * d:].view(torch.bfloat16)
        words[..., 1::2] = least.view(n // 16, 1, 1, 16, 1).expand(-1, -1, -1, -1, d // 64).reshape(n // 16, 1, 1, -1)
    table = torch.arange(n // 16, dtype=torch.int32, device=cuda)[None]
    lens = torch.tensor([n], dtype=torch.int32, device=cuda)
    got = ktt.paged_read(pages[False].to(cuda), pages[True].to(cuda), table, lens)
    for out, value in zip(got, (False, True)):
        code, step, low = (t.double().transpose(1, 2).reshape(n, -1) for t in po.unpack(pages[value], value))
        exact = (low.unsqueeze(-1) + step.unsqueeze(-1) * code.view(n, -1, 64)).reshape(n, d)
        have = out[0, 0].cpu()
        bits = have.view(torch.int16)
        for other in ((bits + 1).view(torch.bfloat16), (bits - 1).view(torch.bfloat16)):     # no neighbour is nearer
            near, far = (have.double() - exact).abs(), (other.double() - exact).abs()
            assert ((near < far) | ((near == far) & (bits & 1 == 0)) | (have == 0)).all()
