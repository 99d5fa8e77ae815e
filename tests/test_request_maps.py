"""Block tables and slot maps built on the GPU (ops/request_maps.py) against
oracle/beam_ref.py and against what the host builds (build_tables, PagedCacheView.reserve):
whole numbers, exact."""
import pytest
import torch

from gpu_utils import graph_replays_match
from oracle.beam_ref import block_tables_ref, slot_map_ref

gpu = pytest.mark.gpu
FIELDS = ((torch.int32, -7), (torch.int64, -7), (torch.int64, -7), (torch.int64, -7), (torch.int32, -7))


def _ops():
    from acorninfer_amd.ops import request_maps
    return request_maps


def test_refusals():
    o = _ops()
    i32 = torch.int32
    b, n = torch.zeros(9, dtype=i32), torch.zeros(3, dtype=i32)
    tab = torch.zeros(3, 4, dtype=i32)
    for bad in (lambda: o.block_tables(b.long(), n, 16, 4), lambda: o.block_tables(b, n.long(), 16, 4),
                lambda: o.block_tables(b, n, 12, 4), lambda: o.block_tables(b, n, 0, 4),
                lambda: o.block_tables(b, n, 16, 0), lambda: o.block_tables(b[None], n, 16, 4),
                lambda: o.block_tables(b[::2], n, 16, 4),
                lambda: o.block_tables(b, n, 16, 4, out=tab[:2]),
                lambda: o.slot_map(tab.long(), n, n, 16, 5), lambda: o.slot_map(tab, n[:2], n, 16, 5),
                lambda: o.slot_map(tab, n, n.long(), 16, 5), lambda: o.slot_map(tab, n, n, 24, 5),
                lambda: o.slot_map(tab, n, n, 16, -1), lambda: o.slot_map(tab[:, :0], n, n, 16, 5),
                lambda: o.slot_map(tab, n, n, 16, 5, out=o.SlotMap(*[n] * 6))):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(ValueError):
        o.block_tables(b, n, 16, 4)
    with pytest.raises(ValueError):
        o.slot_map(tab, n, n, 16, 5)


def test_entries_refuse_without_a_gpu():
    from acorninfer_amd import _lib
    L, p = _lib.lib(), 64
    def tables(T=9, N=3, width=4, P=16, b=p):
        return L.acorn_block_tables(b, T, p, p, N, width, P, 0, None)
    assert tables(T=-1) == tables(N=-1) == tables(width=0) == tables(P=24) == _lib.ERR_SHAPE
    assert tables(P=2**31) == tables(N=2**30) == _lib.ERR_SHAPE
    assert tables(b=None) == _lib.ERR_VALUE and tables(N=0) == 0
    def slots(N=3, R=5, width=4, P=16, t=p, seq=p):
        return L.acorn_slot_map(t, p, p, seq, p, p, p, p, p, N, R, width, P, None)
    assert slots(N=-1) == slots(R=-1) == slots(width=0) == slots(P=0) == _lib.ERR_SHAPE == slots(P=2**31)
    assert slots(t=None) == slots(seq=None) == _lib.ERR_VALUE and slots(N=0) == 0


def _lengths(N, most, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, most + 1, (N,), generator=g).int()


@gpu
@pytest.mark.parametrize("P", [1, 16, 64])
@pytest.mark.parametrize("N,most,width", [(1, 1, 1), (3, 100, 5), (64, 4000, 300), (5, 3000, 2100),
                                          (2500, 90, 7), (5000, 40, 2)])
def test_block_tables(P, N, most, width):
    lengths = _lengths(N, most, N)
    lengths[0] = most
    if N > 3:
        lengths[1], lengths[2] = 0, -5
    total = int((-(-lengths.clamp_min(0).long() // P)).sum())
    g = torch.Generator().manual_seed(P)
    for short in (0, min(3, total)):                          # and a list that ends too early
        blocks = torch.randperm(total + 1, generator=g)[:total - short].int()
        got = _ops().block_tables(blocks.cuda(), lengths.cuda(), P, width, pad=-3)
        assert torch.equal(got.cpu(), block_tables_ref(blocks, lengths, P, width, pad=-3))


@gpu
@pytest.mark.parametrize("P", [1, 16, 64])
@pytest.mark.parametrize("N,count,rows", [(1, 1, 1), (4, 9, None), (64, 1, 64), (3, 700, 900), (7, 300, 9),
                                          (1500, 3, None), (2100, 1, 2200), (2, 5, 0)])
def test_slot_map(P, N, count, rows):
    """Requests that bring nothing, rows behind the last one, rows that are cut off, tokens past the
    table."""
    g = torch.Generator().manual_seed(N)
    starts = torch.randint(0, 200, (N,), generator=g).int()
    counts = torch.randint(0, count + 1, (N,), generator=g).int()
    counts[-1] = count
    if N > 3:
        counts[1], starts[2] = -4, -2
    rows = int(counts.clamp_min(0).sum()) + 11 if rows is None else rows
    W = 6
    tables = torch.randint(0, 999, (N, W), generator=g).int()
    into = [torch.full((rows,), v, dtype=t) for t, v in FIELDS]
    out = _ops().SlotMap(*(t.cuda() for t in into), torch.full((N,), -7).int().cuda())
    got = _ops().slot_map(tables.cuda(), starts.cuda(), counts.cuda(), P, rows, out=out)
    want = slot_map_ref(tables, starts, counts, P, rows, into)
    for name, a, b in zip(got._fields, got, want):
        assert torch.equal(a.cpu(), b), name


@gpu
def test_they_agree_with_the_host():
    from types import SimpleNamespace

    from acorninfer_amd.cache.pager import BlockAllocator, PagedCacheView
    from acorninfer_amd.ops.paged_attention import build_tables
    P, pre, new = 16, [0, 5, 31, 64], [40, 1, 17, 0]
    alloc = BlockAllocator(64)
    cache = SimpleNamespace(allocator=alloc, page_size=P)
    views = [PagedCacheView(cache) for _ in pre]
    targets = []
    for v, a, b in zip(views, pre, new):
        v._grow_to(-(-a // P))
        v._lens[0] = a
        targets += v.reserve(b)
    total = [a + b for a, b in zip(pre, new)]
    want, _ = build_tables(views, P, "cpu", lens_override=total)
    blocks = torch.tensor([x for v in views for x in v.table], dtype=torch.int32).cuda()
    def dev(x):
        return torch.tensor(x, dtype=torch.int32).cuda()
    tables = _ops().block_tables(blocks, dev(total), P, want.shape[1])
    assert torch.equal(tables.cpu(), want)
    got = _ops().slot_map(tables, dev(pre), dev(new), P, sum(new))
    assert list(zip(got.pages.tolist(), got.slots.tolist())) == targets


@gpu
def test_in_a_graph():
    o = _ops()
    lengths = _lengths(70, 500, 1).cuda()
    blocks = torch.arange(70 * 32, device="cuda", dtype=torch.int32)
    out = o.block_tables(blocks, lengths, 16, 32)
    assert graph_replays_match(lambda: o.block_tables(blocks, lengths, 16, 32, out=out), lambda: out)
    rows = int(lengths.sum())
    m = o.slot_map(out, torch.zeros_like(lengths), lengths, 16, rows)
    zero = torch.zeros_like(lengths)
    assert graph_replays_match(lambda: o.slot_map(out, zero, lengths, 16, rows, out=m), lambda: m.pages)


@gpu
@pytest.mark.parametrize("P", [1, 16, 2**30])
def test_positions_at_the_ends_of_their_type(P):
    """The first and the last starts that 32 bits hold: whole numbers of 64 bits, pages of -1."""
    starts = torch.tensor([-2**31, -1, 2**31 - 2, 5]).int()
    counts = torch.tensor([3, 2, 2, 1]).int()
    tables = torch.arange(12).view(4, 3).int()
    into = [torch.full((8,), v, dtype=t) for t, v in FIELDS]
    got = _ops().slot_map(tables.cuda(), starts.cuda(), counts.cuda(), P, 8)
    assert got.positions.tolist() == [-2**31, -2**31 + 1, -2**31 + 2, -1, 0, 2**31 - 2, 2**31 - 1, 5]
    into[4] = into[4].long()                     # (a length of 2^31 stops at 2^31 - 1)
    want = slot_map_ref(tables, starts, counts, P, 8, into)
    want[4] = want[4].clamp_max(2**31 - 1).int()
    for name, a, b in zip(got._fields, got, want):
        assert torch.equal(a.cpu(), b), name
    lengths = torch.tensor([2**31 - 1, -2**31, 1]).int()
    blocks = torch.arange(9).int()
    assert torch.equal(_ops().block_tables(blocks.cuda(), lengths.cuda(), P, 5, pad=-2).cpu(),
                       block_tables_ref(blocks, lengths, P, 5, pad=-2))
