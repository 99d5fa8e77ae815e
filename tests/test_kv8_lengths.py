"""Attention over the 8-bit cache for sequences that fill their last page: lengths past the table
count as the tokens its pages hold."""
import pytest
import torch

gpu = pytest.mark.gpu


def _kv8():
    from acorninfer_amd.ops import kv8
    return kv8


def _sequences(lens, KV, D, P, dtype, g):
    """Sequences in blocks anywhere; every byte that is no token's is NaN."""
    need = [-(-n // P) for n in lens]
    NB = sum(need) + 3
    perm = torch.randperm(NB, generator=g)
    tables = torch.full((len(lens), max(need)), 1 << 30, dtype=torch.int32)
    first = 0
    for i, n in enumerate(need):
        tables[i, :n] = perm[first:first + n]
        first += n
    kv = _kv8().KV8Pages(*(torch.full((NB, KV, P // 16, n), b, dtype=torch.uint8, device="cuda")
                           for n, b in ((16 * D, 0x7F), (16 * D, 0xFF), (32, 255))))
    pages = torch.cat([tables[i].long()[torch.arange(n) // P] for i, n in enumerate(lens)])
    slots = torch.cat([torch.arange(n) % P for n in lens])
    k, v = (torch.randn(len(pages), KV, D, generator=g).to(dtype).cuda() for _ in range(2))
    _kv8().kv8_scatter(k, v, kv, pages.cuda(), slots.cuda())
    return kv, tables


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S", [1, 3, 40, None])
def test_a_length_past_the_table_counts_the_tables_tokens(S, dtype):
    """608 tokens fill 38 pages: any greater length is that one, bit for bit, and finite; the other
    sequence keeps its bits. (Every byte past the pages' tokens is NaN.)"""
    H, KV, D, P = 8, 2, 128, 16
    g = torch.Generator().manual_seed(4)
    kv, tables = _sequences([608, 40], KV, D, P, dtype, g)
    assert tables.shape[1] * P == 608
    q = torch.randn(2, H, D, generator=g).to(dtype).cuda()

    def run(a):
        lens = torch.tensor([a, 40], dtype=torch.int32, device="cuda")
        return _kv8().paged_decode_attention_kv8(q, kv, tables.cuda(), lens, S)
    good = run(608)
    assert torch.isfinite(good).all()
    for n in (609, 1 << 20, 1 << 30, (1 << 31) - 1):
        assert torch.equal(run(n), good), n
    shorter = run(607)
    assert torch.isfinite(shorter).all() and not torch.equal(shorter[0], good[0])
    assert torch.equal(shorter[1], good[1])
    assert torch.isnan(run(0)[0]).all() and torch.isnan(run(-5)[0]).all()


@gpu
@pytest.mark.parametrize("m", [4, 40])
def test_a_windows_length_past_the_table_counts_the_tables_tokens(m):
    H, KV, D, P = 8, 2, 128, 16
    g = torch.Generator().manual_seed(4)
    kv, tables = _sequences([608, 60], KV, D, P, torch.bfloat16, g)
    q = torch.randn(2, m, H, D, generator=g).bfloat16().cuda()

    def run(a):
        return _kv8().paged_verify_attention_kv8(q, kv, tables.cuda(),
                                                 torch.tensor([a, 60], dtype=torch.int32, device="cuda"))
    good = run(608)
    assert torch.isfinite(good).all()
    for n in (609, 1 << 30, (1 << 31) - 1):
        assert torch.equal(run(n), good), n
