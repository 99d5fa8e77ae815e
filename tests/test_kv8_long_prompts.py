"""Long prompts over the 8-bit cache, every row and head against decode over the same cache, by a bound
that a lost or doubled step of 32 keys misses."""
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


LOST = 4 * 2.0 ** -8                     # of a row's norm


def test_a_lost_step_of_keys_shows_in_a_rows_norm():
    """CPU: softmax over 5000 tokens whose scores spread by 1 at most, as in the next test, without
    32 of them or with 32 of them twice, is off by more than the bound that test holds rows to; with
    its weights rounded to bf16, by far less. (At a spread of 2 few tokens hold the weight, and 32
    others may not show.)"""
    g = torch.Generator().manual_seed(1)
    v = torch.randn(5000, 128, generator=g).double()
    for spread in (0.5, 1.0):
        p = torch.exp(spread * torch.randn(5000, generator=g)).double()
        want = p @ v / p.sum()
        q = p.float().bfloat16().double()
        assert (q @ v / q.sum() - want).norm() < 0.5 * LOST * want.norm()
        for first in (0, 1600, 4960):
            for factor in (0.0, 2.0):
                bad = p.clone()
                bad[first:first + 32] *= factor
                assert (bad @ v / bad.sum() - want).norm() > 1.5 * LOST * want.norm()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,KV,D,segs", [(8, 2, 128, [(0, 5000)]), (8, 8, 64, [(900, 1500), (0, 700)])])
def test_prompt_rows_equal_decode_rows(H, KV, D, segs, dtype):
    """Every row and head of long prompts against decode over the same cache, by the norm of the
    head's output. v has independent signs, so a weight's rounding (u at most, each its own) moves
    the output by u of its norm, give or take; the two results' roundings and their 32-bit steps by
    as much again; 4 u of bf16 holds both types."""
    P = 16
    g = torch.Generator().manual_seed(21)
    kv, tables = _sequences([a + b for a, b in segs], KV, D, P, dtype, g)
    R = sum(n for _, n in segs)
    q = torch.randn(R, H, D, generator=g).to(dtype).cuda()
    row0 = torch.tensor([0] + [n for _, n in segs[:-1]]).cumsum(0).int().cuda()
    pos0, nq = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in zip(*segs))
    out = _kv8().paged_prefill_attention_kv8(q, kv, tables.cuda(), row0, pos0, nq, max(n for _, n in segs))
    at = 0
    for i, (a, n) in enumerate(segs):
        lens = torch.arange(a + 1, a + n + 1, dtype=torch.int32, device="cuda")
        dec = _kv8().paged_decode_attention_kv8(q[at:at + n], kv, tables[i:i + 1].cuda().expand(n, -1).contiguous(),
                                                lens, 1).double()
        off = (out[at:at + n].double() - dec).norm(dim=-1) / dec.norm(dim=-1)
        assert float(off.max()) <= LOST, (i, int(off.amax(-1).argmax()), float(off.max()))
        at += n
