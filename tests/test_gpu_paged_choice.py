"""Which way attention over pages takes, on both sides of each line of the choice, with the result against float64: the pass over
pages counts as a decode call, the tensor path as a flash one."""

import pytest
import torch

import kohaku_tt_b200 as ktt
from tests.launched import launched
from tests.test_gpu_paged import _cache, _check, _x

pytestmark = pytest.mark.gpu

BITS = [16, 4]


def _takes(cuda, bits, tensor, *args, calls=1, **kw):
    """_check, and whether the call went over the tensor path (and in how many launches of the forward)."""
    before = ktt.counters()
    _check(cuda, bits, *args, dense_four_bits=tensor and bits == 4, **kw)
    after = ktt.counters()
    got = {name: after[name] - before[name] for name in ("attention_decode", "attention_flash")}
    assert got == {"attention_decode": 0 if tensor else 1, "attention_flash": calls if tensor else 0}


def _merges(cuda, bits, d, h, hk, page, n, lengths, causal):
    """Whether a dense call's keys are cut into parts."""
    kp, vp, table = _cache(bits, d, hk, page, lengths)
    args = (_x(len(lengths), h, n, d).to(cuda), kp.to(cuda), vp.to(cuda), table.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda))
    return any("merge_parts" in x.name for x in launched(lambda: ktt.sdpa_paged(*args, is_causal=causal)))


# Room for 8,192 keys, three sequences: where the pass over 16 rows of a K / V head, once for each, starts to cost more than dense
# rows and their tiles. D, H, Hk, bits, the most tokens that the pass is for.
LINES = [(64, 6, 2, 16, 32), (64, 6, 2, 4, 42), (128, 16, 2, 16, 20), (128, 16, 2, 4, 22), (64, 3, 3, 16, 64), (64, 3, 3, 4, 64)]


@pytest.mark.parametrize("d,h,hk,bits,most", LINES)
@pytest.mark.parametrize("beyond", [0, 1])
def test_both_sides_of_the_cost(cuda, d, h, hk, bits, most, beyond):
    _takes(cuda, bits, bool(beyond), d, h, hk, 32, most + beyond, [60, 300, 1], wide=256)
    _takes(cuda, bits, bool(beyond), d, h, hk, 32, [most + beyond, 1, 0], [60, 300, 1], wide=256, packed=True, max_q=most + beyond)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [64, 65])
def test_few_keys_go_by_tokens(cuda, bits, d, n):
    _takes(cuda, bits, n == 65, d, 6, 2, 16, n, [60, 100])


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("d,causal", [(64, True), (64, False), (128, True), (128, False)])
def test_dense_chunks_with_few_keys_or_none(cuda, bits, d, causal):
    """Sequences without a key, with fewer keys than queries, and that end on a tile's last key."""
    _takes(cuda, bits, True, d, 6, 3, 16, 70, [0, 3, 70, 128], causal=causal)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("d,causal", [(64, True), (64, False), (128, True), (128, False)])
def test_dense_chunks_that_are_cut(cuda, bits, d, causal):
    """A sequence without a key beside one that is cut; as many queries as keys."""
    for h, hk, page, n, lengths in ((3, 3, 16, 70, [0, 2500]), (2, 1, 64, 1100, [3000])):
        assert _merges(cuda, bits, d, h, hk, page, n, lengths, causal)
        _takes(cuda, bits, True, d, h, hk, page, n, lengths, causal=causal, seed=4)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("d,hk", [(128, 8), (64, 16)])
def test_dense_chunks_over_more_room_than_one_launch_takes(cuda, bits, d, hk):
    """Room for 65,536 keys: the dense rows of 4 sequences are 1 GB, so 6 are two launches of 4 and 2."""
    _takes(cuda, bits, True, d, hk, hk, 64, 66, [100, 49, 3, 257, 0, 64], wide=1024, calls=2)


@pytest.mark.parametrize("n", [66, 130])
def test_pages_and_queries_in_other_orders(cuda, n):
    """The tensor path's reading of bf16 pages stored [pages, page, Hk, D], keys and values in one storage: the same bits."""
    d, h, hk, page, lengths = 128, 8, 2, 16, [175, 140]
    kp, vp, table = _cache(16, d, hk, page, lengths)
    lens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    q = _x(2, h, n, d, seed=4).to(cuda)
    both = torch.stack([kp.transpose(1, 2), vp.transpose(1, 2)], dim=1).to(cuda)
    want = ktt.sdpa_paged(q, kp.to(cuda), vp.to(cuda), table.to(cuda), lens)
    got = ktt.sdpa_paged(q.transpose(1, 2).contiguous().transpose(1, 2), both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), table.to(cuda), lens)
    assert torch.equal(got, want)


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("d", [64, 128])
def test_a_process_s_first_chunk_inside_a_capture(cuda, bits, d):
    """Chunks that are cut and whole, captured before any call has run; then two replays at once with calls on a third stream."""
    import subprocess
    import sys

    code = f"""
import torch, kohaku_tt_b200 as ktt
dev = torch.device("cuda:0")
kp, vp = ktt.paged_cache(188, 2, 16, {d}, bits={bits}, device=dev)
table = torch.arange(188, dtype=torch.int32, device=dev).view(2, 94)
zero, lens = torch.zeros(2, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
k, v = (torch.randn(2, 2, 1500, {d}, device=dev).bfloat16() for _ in range(2))
qs = [torch.randn(2, h, 140, {d}, device=dev).bfloat16() for h in (2, 16)]
torch.cuda.synchronize()
graphs, got = [], []
for q in qs:
    graphs.append(torch.cuda.CUDAGraph())
    with torch.cuda.graph(graphs[-1]):
        ktt.paged_append(k, v, kp, vp, table, zero, lengths_out=lens)
        got.append(ktt.sdpa_paged(q, kp, vp, table, lens))
for g in graphs:
    g.replay()
torch.cuda.synchronize()
assert lens.tolist() == [1500, 1500]
want = [ktt.sdpa_paged(q, kp, vp, table, lens) for q in qs]
streams = [torch.cuda.Stream() for _ in range(3)]
for _ in range(5):
    torch.cuda.synchronize()
    for s, g in zip(streams, graphs):
        with torch.cuda.stream(s):
            g.replay()
    with torch.cuda.stream(streams[2]):
        eager = [ktt.sdpa_paged(q, kp, vp, table, lens) for q in qs]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(c, b) and b.isfinite().all() for a, b, c in zip(got, want, eager))
print("same")
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stdout + done.stderr[-3000:]
