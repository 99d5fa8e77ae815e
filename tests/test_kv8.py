"""The 8-bit paged KV cache (ops/kv8.py): writing, reading back, the qkv epilogue and attention
against oracle/kv8_ref.py (64 bits). Bytes, codes and values read back are exact. Attention is
held, element by element, to the bound oracle.kv8_ref.tolerance derives from the roundings the
kernels make."""
import ctypes
import math

import numpy as np
import pytest
import torch

from gpu_utils import graph_replays_match
from oracle.kv8_ref import E4M3, Pool, attend, quantise_row, scale_exp, tolerance

gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def _kv8():
    from acorninfer_amd.ops import kv8
    return kv8


# ---- CPU: the oracle, the planner and the refusals -------------------------------------------


def test_format_of_the_oracle():
    assert E4M3[0x7E] == 448 and E4M3[1] == 2.0 ** -9 and math.isnan(E4M3[0x7F])
    for amax, e in ((448.0, 0), (448.1, 1), (224.0, -1), (1.75, -8), (1.76, -7), (0.0, -126),
                    (2.0 ** -149, -126), (3.0e38, 120)):
        assert scale_exp(amax) == e, amax
    g = torch.Generator().manual_seed(0)
    x = torch.randn(200, 64, generator=g).double().numpy() * 10.0 ** np.linspace(-30, 30, 200)[:, None]
    for row in x:
        b, code, ok = quantise_row(row, False)
        y = E4M3[b] * 2.0 ** (code - 127)
        assert ok and (np.abs(y - row) <= 2.0 ** -4 * np.abs(row) + 2.0 ** (code - 127 - 10)).all()
        # torch's own rounding to the type agrees, byte by byte
        t = torch.from_numpy(row * 2.0 ** (127 - code)).float().to(torch.float8_e4m3fn)
        assert np.array_equal(t.view(torch.uint8).numpy(), b)
    assert quantise_row(np.array([1.0, math.inf]), False)[1] == 255
    assert E4M3[quantise_row(np.array([65504.0]), True)[0][0]] * 256 == 61440


def test_oracle_notices_a_planted_mistake():
    """Attention over the oracle's own values with one token's scale doubled is out of tolerance."""
    g = torch.Generator().manual_seed(1)
    pool = Pool(2, 1, 64, 16)
    k, v = torch.randn(2, 20, 1, 64, generator=g)
    at = torch.arange(20)
    pool.put(k, v, at // 16, at % 16)
    q = torch.randn(2, 64, generator=g)
    good, mean, big = attend(q, *pool.values([0, 1], range(20)))
    pool.scales[0, 0, 0, 16 + 5] += 1
    bad, _, _ = attend(q, *pool.values([0, 1], range(20)))
    assert ((bad - good).abs() > tolerance(good, mean, big, torch.bfloat16, 20)).any()


@pytest.mark.parametrize("batch,kv,pages,P", [(1, 1, 1, 16), (1, 8, 8190, 16), (64, 8, 512, 16),
                                              (8, 8, 40, 32), (0, 8, 1, 16), (300, 8, 4000, 16)])
def test_split_rule(batch, kv, pages, P):
    s = _kv8().kv8_splits(batch, kv, pages, P)
    assert 1 <= s <= max(1, pages)


def test_split_rule_keeps_to_the_table():
    """Whole pages of any size, and never more splits than pages."""
    rule = _kv8().kv8_splits
    for P in (16, 32, 1024, 65536):
        for pages in (1, 2, 3, 31, 64, 65, 500, 9000):
            for batch in (1, 2, 7, 12, 31, 33, 200):
                for kv in (1, 5, 8):
                    assert 1 <= rule(batch, kv, pages, P) <= pages, (batch, kv, pages, P)


def test_shapes_supported():
    k = _kv8()
    assert k.kv8_supported(128, 16) and k.kv8_supported(64, 64)
    for D, P in ((96, 16), (256, 16), (128, 8), (128, 48), (128, 0), (128, 131072)):
        assert not k.kv8_supported(D, P)
        with pytest.raises(NotImplementedError):
            k.kv8_pages(2, 1, D, P, "cpu")
    ok = k.kv8_attention_supported
    assert ok(torch.bfloat16, 128, 16, 32, 8) and not ok(torch.float32, 128, 16, 32, 8)
    assert not ok(torch.bfloat16, 128, 16, 24, 8) and not ok(torch.bfloat16, 128, 16, 9, 8)


def test_cpu_tensors_are_refused():
    k = _kv8()
    kv = k.kv8_pages(4, 2, 64, 16, "cpu")
    i64 = torch.zeros(1, dtype=torch.int64)
    i32 = torch.ones(1, dtype=torch.int32)
    tab = torch.zeros(1, 1, dtype=torch.int32)
    row = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        k.kv8_scatter(row, row, kv, i64, i64)
    with pytest.raises(ValueError):
        k.kv8_gather(kv, tab, i32, i32, i32, 1, 1)
    with pytest.raises(ValueError):
        k.qkv_norm_rope_kv8(torch.zeros(1, 6 * 64, dtype=torch.bfloat16), kv, i64, i64, i64,
                            torch.ones(32), w, w, 1e-6, 2)
    with pytest.raises(ValueError):
        k.paged_decode_attention_kv8(row, kv, tab, i32)
    with pytest.raises(ValueError):
        k.paged_prefill_attention_kv8(row, kv, tab, i32, i32, i32, 1)
    with pytest.raises(ValueError):
        k.paged_verify_attention_kv8(torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16), kv, tab, i32)


def test_c_entries_refuse_before_any_launch():
    """Shapes, types and pointers are checked on the host: no GPU is needed to be refused."""
    from acorninfer_amd import _lib
    L = _lib.lib()
    SH, DT, VA, UN = _lib.ERR_SHAPE, _lib.ERR_DTYPE, _lib.ERR_VALUE, _lib.ERR_UNSUPPORTED
    p = 64                                            # a pointer that is never followed

    def scatter(rows=1, KV=2, D=64, P=16, NB=4, dt=2, k=p, tiles=p, rs=128):
        return L.acorn_kv8_scatter(k, p, tiles, p, p, p, p, rows, KV, D, P, NB, rs, 64, rs, 64, dt, None)
    assert scatter(rows=0) == 0
    assert [scatter(rows=-1), scatter(KV=0), scatter(P=24), scatter(P=8), scatter(NB=0)] == [SH] * 5
    assert [scatter(D=96), scatter(D=256)] == [UN] * 2
    assert [scatter(k=None), scatter(k=66), scatter(tiles=72), scatter(rs=65)] == [VA] * 4
    assert scatter(dt=7) == DT

    def gather(N=1, R=1, M=1, KV=2, D=64, P=16, W=1, out=p, dt=2):
        return L.acorn_kv8_gather(p, p, p, p, p, p, p, out, p, N, R, M, KV, D, P, 4, W, dt, None)
    assert gather(N=0) == gather(R=0) == gather(M=0) == 0
    assert [gather(N=-1), gather(W=0), gather(P=0), gather(R=-1), gather(W=1 << 30)] == [SH] * 5
    assert [gather(out=None), gather(out=72), gather(dt=9), gather(D=32)] == [VA, VA, DT, UN]

    def qkv(ns=1, rows=1, H=2, KV=2, D=64, P=16, dt=2, part=p):
        return L.acorn_qkv_epilogue_kv8(part, ns, p, p, p, p, p, p, rows, H, KV, D, P, 4, p, p, 1e-6,
                                        p, p, dt, None)
    assert qkv(rows=0) == 0
    assert [qkv(ns=-1), qkv(H=0), qkv(KV=0)] == [SH] * 3
    assert [qkv(part=None), qkv(part=72), qkv(dt=0), qkv(D=80)] == [VA, VA, DT, UN]

    def decode(B=1, H=2, KV=2, D=64, P=16, W=1, S=1, dt=2, q=p, ws=p):
        return L.acorn_paged_attention_kv8(q, p, p, p, p, p, p, ws, p, B, H, KV, D, P, 4, W, S, 0.1, dt,
                                           None)
    assert decode(B=0) == 0
    assert [decode(H=3), decode(W=0), decode(S=0), decode(P=48), decode(B=70000)] == [SH] * 5
    assert [decode(D=32), decode(H=6), decode(H=32)] == [UN] * 3
    assert [decode(q=None), decode(S=2, ws=None), decode(q=72)] == [VA] * 3
    assert decode(dt=0) == DT

    def prefill(N=1, R=1, M=1, H=2, row0=p, nq=p, ws=None, dt=2, W=1):
        return L.acorn_paged_prefill_attention_kv8(p, p, p, p, p, row0, p, nq, p, N, R, M, H, 2, 64, 16,
                                                   4, W, 0.1, dt, ws, 0, None)
    assert prefill(N=0) == prefill(R=0) == prefill(M=0) == 0
    assert [prefill(H=3), prefill(W=0), prefill(row0=None, nq=None, R=3)] == [SH] * 3
    assert [prefill(row0=None), prefill(nq=None), prefill(ws=72)] == [VA] * 3
    assert [prefill(H=6), prefill(dt=0)] == [UN, DT]
    n = ctypes.c_int64(-1)
    assert L.acorn_paged_prefill_workspace_kv8(1, 5, 5, 32, 8, 128, 16, 500, ctypes.byref(n)) == 0
    assert n.value > 0
    assert L.acorn_paged_prefill_workspace_kv8(1, 5, 5, 32, 8, 128, 16, 500, None) == VA


# ---- GPU: writing and reading back -----------------------------------------------------------


def _rows(R, KV, D, dtype, seed, spread=6):
    """Rows over many magnitudes, with zeros, signed zeros and rows at the borders of a scale."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, KV, D, generator=g)
    x *= 10.0 ** (torch.rand(R, KV, 1, generator=g) * 2 * spread - spread)
    x[torch.rand(R, KV, D, generator=g) < 0.05] = -0.0
    flat = x.view(R * KV, D)
    for i, v in enumerate((0.0, 448.0, 449.0, 1.75, 1.7578125, -3.5, 2.0 ** -14)):
        if i < R * KV:
            flat[i] = v * (1 if i % 2 else -1) * torch.rand(D, generator=g)
            flat[i, i % D] = v
    return x.to(dtype)


def _to_gpu(pool):
    return _kv8().KV8Pages(*(torch.from_numpy(x).cuda() for x in (pool.k, pool.v, pool.scales)))


def _same_bytes(kv, pool):
    for a, b in zip(kv, (pool.k, pool.v, pool.scales)):
        assert np.array_equal(a.cpu().numpy(), b)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("KV,D,P,R", [(1, 64, 16, 1), (8, 128, 16, 19), (5, 128, 32, 70), (2, 64, 64, 33)])
def test_scatter_writes_the_oracles_bytes(dtype, KV, D, P, R):
    """Every byte of the pool: the rows' own as the oracle's, all others as they were."""
    g = torch.Generator().manual_seed(R)
    pool = Pool(R // P + 4, KV, D, P)
    pool.k[:] = 3
    pool.scales[:] = 77
    kv = _to_gpu(pool)
    spread = 3 if dtype == torch.float16 else 25 if dtype == torch.bfloat16 else 30
    k, v = _rows(R, KV, D, dtype, 2 * R, spread), _rows(R, KV, D, dtype, 2 * R + 1, spread)
    at = torch.randperm(pool.NB * P, generator=g)[:R]
    pages, slots = at // P, at % P
    pool.put(k, v, pages, slots, dtype == torch.float16)
    _kv8().kv8_scatter(k.cuda(), v.cuda(), kv, pages.cuda(), slots.cuda())
    _same_bytes(kv, pool)


@gpu
def test_scatter_takes_strided_rows():
    """k and v as slices of one projection's output, transposed, with dims not side by side, from
    an odd address."""
    R, KV, D, P = 21, 4, 128, 16
    g = torch.Generator().manual_seed(3)
    base = torch.randn(R, 3 * KV * D + 8, generator=g).bfloat16().cuda()
    k, v = base[:, KV * D:2 * KV * D].view(R, KV, D), base[:, 2 * KV * D:3 * KV * D].view(R, KV, D)
    forms = [(k, v), (k.transpose(0, 1).contiguous().transpose(0, 1), v),
             (k.transpose(1, 2).contiguous().transpose(1, 2), v.expand(R, KV, D)),
             (base[:, 3:3 + KV * D].view(R, KV, D), v), (k[:, :1].expand(R, KV, D), v)]
    at = torch.arange(R)
    for a, b in forms:
        pool = Pool(3, KV, D, P)
        kv = _to_gpu(pool)
        pool.put(a.cpu(), b.cpu(), at // P, at % P)
        _kv8().kv8_scatter(a, b, kv, (at // P).cuda(), (at % P).cuda())
        _same_bytes(kv, pool)


@gpu
def test_scatter_of_rows_that_are_not_finite_and_of_targets_outside():
    """An infinity or NaN in k or v makes that (token, head) NaN and no other; targets outside the
    pool are skipped; fp16's largest numbers stay finite in fp16."""
    R, KV, D, P = 9, 3, 64, 16
    k, v = _rows(R, KV, D, torch.float16, 5, 2), _rows(R, KV, D, torch.float16, 6, 2)
    k[1, 0, 5], v[2, 1, 63], k[3, 2, 0], v[4, 0, 1] = math.inf, -math.inf, math.nan, 65504.0
    k[5, 1, 2], k[5, 1, 3] = -65504.0, 63456.0
    pages = torch.tensor([0, 1, 2, 0, 1, 2, -1, 3, 1])
    slots = torch.tensor([0, 1, 2, 3, 15, 14, 0, 0, 16])
    pool = Pool(3, KV, D, P)
    kv = _to_gpu(pool)
    pool.put(k, v, pages, slots, True)
    _kv8().kv8_scatter(k.cuda(), v.cuda(), kv, pages.cuda(), slots.cuda())
    _same_bytes(kv, pool)
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    tab = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
    gk, gv = _kv8().kv8_gather(kv, tab, 0 * one, 0 * one, 48 * one, 48, 48, dtype=torch.float16)
    for t, h in ((17, 0), (34, 1), (3, 2)):
        assert torch.isnan(gk[t, h]).all() and torch.isnan(gv[t, h]).all()
    assert int(torch.isnan(gk).sum()) == int(torch.isnan(gv).sum()) == 3 * D
    assert not torch.isinf(gk).any() and not torch.isinf(gv).any()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("KV,D,P", [(8, 128, 16), (3, 64, 32)])
def test_gather_reads_the_oracles_values(dtype, KV, D, P):
    """Runs from any token of sequences of any length, packed with gaps: the rows as rounded once
    from 64 bits, the gaps left as they were, rows past R or the table not written."""
    g = torch.Generator().manual_seed(8)
    pool = Pool(12, KV, D, P)
    n = pool.NB * P
    at = torch.randperm(n, generator=g)
    pool.put(_rows(n, KV, D, torch.float16, 9, 2), _rows(n, KV, D, torch.float16, 10, 2), at // P, at % P, True)
    kv = _to_gpu(pool)
    tables = torch.stack([torch.randperm(12, generator=g)[:5] for _ in range(5)]).int()
    runs = [(0, 1), (7, 30), (16, 16), (3, 0), (5 * P - 9, 20)]          # the last leaves its table
    row0, r = [], 2
    for _, m in runs:
        row0.append(r)
        r += m + 2
    R = r - 6
    meta = [torch.tensor(x, dtype=torch.int32) for x in (row0, [a for a, _ in runs], [m for _, m in runs])]
    want = [torch.full((R, KV, D), 7.0, dtype=dtype) for _ in range(2)]
    for i, (p0, m) in enumerate(runs):
        m = min(m, 5 * P - p0, R - row0[i])
        if m > 0:
            for w, x in zip(want, pool.values(tables[i], range(p0, p0 + m))):
                w[row0[i]:row0[i] + m] = x.to(dtype)
    out = tuple(torch.full((R, KV, D), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    got = _kv8().kv8_gather(kv, tables.cuda(), *(m.cuda() for m in meta), 30, R, dtype=dtype, out=out)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


# ---- GPU: the qkv epilogue -------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,D,P,R,S", [(32, 8, 128, 16, 8, 3), (16, 8, 128, 16, 33, 0), (4, 4, 64, 32, 1, 1),
                                          (20, 5, 64, 16, 5, 9), (64, 8, 128, 16, 3, 0)])
def test_qkv_epilogue(dtype, H, KV, D, P, R, S):
    """q within its one rounding and the 32-bit arithmetic before it; k and v within a rounding to
    e4m3; far positions (the angle's product has its own rounding at 2^17)."""
    g = torch.Generator().manual_seed(H + R)
    width = (H + 2 * KV) * D
    x = torch.randn(*((S, R, width) if S else (R, width)), generator=g) * 0.7
    x = x if S else x.to(dtype)
    pos = torch.randint(0, 131072, (R,), generator=g)
    pos[0] = 0
    inv_freq = 1.0 / 1e6 ** (torch.arange(0, D, 2).float() / D)
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(dtype) for _ in range(2))
    pool = Pool(R // P + 3, KV, D, P)
    kv = _to_gpu(pool)
    at = torch.randperm(pool.NB * P, generator=g)[:R]
    q = _kv8().qkv_norm_rope_kv8(*[x.cuda(), kv, (at // P).cuda(), (at % P).cuda(), pos.cuda(),
                                   inv_freq.cuda(), qw.cuda(), kw.cuda(), 1e-6, H])
    y = x.double()
    mag = (y.abs().sum(0) if S else y.abs()).view(R, H + 2 * KV, D)
    y = (y.sum(0) if S else y).view(R, H + 2 * KV, D)
    w = torch.cat([qw.double().expand(H, D), kw.double().expand(KV, D)])
    inv = 1 / (y[:, :H + KV].square().mean(-1, keepdim=True) + 1e-6).sqrt()
    z, mag_z = y[:, :H + KV] * inv * w, mag[:, :H + KV] * inv * w.abs()
    ang = pos.double()[:, None, None] * inv_freq.double()
    a, b = z.chunk(2, -1)
    rot = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)
    # 32-bit steps: the planes, the mean square over 128, the root, two products, cos and sin
    # (under 4 ulp with their remainder), the sum: under 64 of 2^-24 of the magnitudes
    ma, mb = mag_z.chunk(2, -1)
    eps = 64 * 2.0 ** -24 * torch.cat([ma + mb, ma + mb], -1)
    u = torch.finfo(dtype).eps / 2
    assert ((q.cpu().double() - rot[:, :H]).abs() <= u * (rot[:, :H].abs() + eps[:, :H]) + eps[:, :H] + 2.0 ** -25).all()
    held = Pool.of(kv, P)
    table = np.arange(pool.NB)
    gk, gv = held.values(table, at)
    vmag = 64 * 2.0 ** -24 * mag[:, H + KV:]
    for got, want, e in ((gk, rot[:, H:], eps[:, H:]), (gv, y[:, H + KV:], vmag)):
        top = (want.abs() + e).amax(-1, keepdim=True)
        grid = 2.0 ** (torch.floor(torch.log2(top)) - 7)           # 2^e at most
        assert ((got - want).abs() <= 2.0 ** -4 * (want.abs() + e) + 2.0 ** -10 * grid + e).all()
        exact = torch.from_numpy(np.stack([[E4M3[quantise_row(r, dtype == torch.float16)[0]] *
                                            2.0 ** (quantise_row(r, dtype == torch.float16)[1] - 127)
                                            for r in rows] for rows in want.numpy()]))
        # (bytes differ only where 64 and 32 bits fall on two sides of a border)
        assert (got == exact).double().mean() > 0.999
    # nothing else was written
    keep = torch.ones(pool.NB * P, dtype=torch.bool)
    keep[at] = False
    rest = torch.arange(pool.NB * P)[keep]
    assert all((x == 0).all() for x in held.values(table, rest))


# ---- GPU: decode attention -------------------------------------------------------------------


def _filled(lens, KV, D, P, dtype, seed, extra=3, junk=True):
    """A pool with sequences of `lens` tokens in blocks anywhere; the rest of the pool, the slots
    behind the last tokens and the table entries behind the last blocks hold what must not matter
    (NaN bytes, NaN codes, block ids outside the pool)."""
    g = torch.Generator().manual_seed(seed)
    need = [max(1, -(-n // P)) for n in lens]
    pool = Pool(sum(need) + extra, KV, D, P)
    if junk:
        pool.k[:], pool.v[:], pool.scales[:] = 0x7F, 0xFF, 255
    perm = torch.randperm(pool.NB, generator=g)
    W = max(need)
    tables = torch.full((len(lens), W), 1 << 30, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = perm[at:at + n]
        at += n
    kv = None
    pages = torch.cat([tables[i].long()[torch.arange(n) // P] for i, n in enumerate(lens)])
    slots = torch.cat([torch.arange(n) % P for n in lens])
    R = len(pages)
    k = (torch.randn(R, KV, D, generator=g) * torch.exp(0.5 * torch.randn(1, 1, D, generator=g))).to(dtype)
    v = (torch.randn(R, KV, D, generator=g) * torch.exp(torch.randn(R, KV, 1, generator=g))).to(dtype)
    kv = _to_gpu(pool)
    if R:
        _kv8().kv8_scatter(k.cuda(), v.cuda(), kv, pages.cuda(), slots.cuda())
    return kv, tables, g


def _check_rows(out, q, pool, tables, seen, dtype):
    """out, q [rows, H, D]; row i sees the first seen[i][1] tokens of table seen[i][0]."""
    held = {}
    worst = 0.0
    for i, (n, L) in enumerate(seen):
        if n not in held or len(held[n][0]) < L:
            held[n] = pool.values(tables[n], range(max(l for m, l in seen if m == n)))
        k, v = held[n]
        want, mean, big = attend(q[i], k[:L], v[:L])
        tol = tolerance(want, mean, big, dtype, L)
        err = (out[i].double() - want).abs()
        assert (err <= tol).all(), f"row {i} over {L} tokens: {(err / tol).max():.2f} of the bound"
        worst = max(worst, float((err / tol).max()))
    return worst


DECODE = [
    # (H, KV, D, P, lens)
    (32, 8, 128, 16, [1]),
    (32, 8, 128, 16, [16, 1, 17, 15, 33, 31, 32]),
    (16, 8, 128, 16, [333]),
    (8, 8, 64, 32, [1, 64, 65, 700]),
    (64, 8, 128, 64, [257, 40]),
    (20, 5, 64, 16, [600, 1, 255]),
    (32, 8, 128, 16, [1500, 90]),
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [None, 1, 2, 5, 64])
@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decode(case, S, dtype):
    H, KV, D, P, lens = DECODE[case]
    kv, tables, g = _filled(lens, KV, D, P, dtype, 30 + case)
    q = (1.5 * torch.randn(len(lens), H, D, generator=g)).to(dtype)
    out = _kv8().paged_decode_attention_kv8(q.cuda(), kv, tables.cuda(),
                                            torch.tensor(lens, dtype=torch.int32).cuda(), S)
    _check_rows(out.cpu(), q, Pool.of(kv, P), tables, [(i, L) for i, L in enumerate(lens)], dtype)


@gpu
@pytest.mark.parametrize("S", [1, 4])
def test_decode_of_peaked_and_rising_scores(S):
    """Scores that rise with the position (the running maximum moves all the way), and one token
    that takes all the weight."""
    H, KV, D, P, L = 4, 1, 128, 16, 700
    pool = Pool(45, KV, D, P)
    kv = _to_gpu(pool)
    g = torch.Generator().manual_seed(2)
    k = torch.zeros(L, KV, D)
    k[:, 0, 0] = torch.linspace(-60, 60, L)
    k[333, 0, 1] = 200.0
    v = torch.randn(L, KV, D, generator=g)
    at = torch.arange(L)
    _kv8().kv8_scatter(k.bfloat16().cuda(), v.bfloat16().cuda(), kv, (at // P).cuda(), (at % P).cuda())
    q = torch.zeros(1, H, D)
    q[0, 0, 0], q[0, 1, 0], q[0, 2, 1], q[0, 3] = 8.0, -8.0, 16.0, 0.0
    q = q.bfloat16()
    tables = torch.arange(45, dtype=torch.int32)[None]
    out = _kv8().paged_decode_attention_kv8(q.cuda(), kv, tables.cuda(),
                                            torch.tensor([L], dtype=torch.int32).cuda(), S)
    _check_rows(out.cpu(), q, Pool.of(kv, P), tables, [(0, L)], torch.bfloat16)


@gpu
@pytest.mark.parametrize("lost", [(0, 64), (0, 470), (300, 600), (40, 41)])
@pytest.mark.parametrize("S", [1, 3, 40, "prefill"])
def test_scores_past_32_bits_have_no_weight(S, lost):
    """Tokens whose products with q pass the least 32-bit number score -inf: the result is that
    of the others, also where a wave, a split or a run of keys holds nothing else."""
    H, KV, D, P, L = 8, 2, 128, 16, 600
    kv, tables, g = _filled([L], KV, D, P, torch.bfloat16, 9)
    at = torch.arange(*lost)
    k = torch.zeros(len(at), KV, D)
    k[:, :, 5] = -3e38
    v = torch.randn(len(at), KV, D, generator=g)
    _kv8().kv8_scatter(k.bfloat16().cuda(), v.bfloat16().cuda(), kv, tables[0].long()[at // P].cuda(),
                       (at % P).cuda())
    q = torch.randn(1, H, D, generator=g)
    q[:, :, 5] = 8.0
    q = q.bfloat16()
    if S == "prefill":
        meta = [torch.tensor([x], dtype=torch.int32).cuda() for x in (0, L - 1, 1)]
        out = _kv8().paged_prefill_attention_kv8(q.cuda(), kv, tables.cuda(), *meta, 1)
    else:
        out = _kv8().paged_decode_attention_kv8(q.cuda(), kv, tables.cuda(),
                                                torch.tensor([L], dtype=torch.int32).cuda(), S)
    rest = [t for t in range(L) if not lost[0] <= t < lost[1]]
    k, v = Pool.of(kv, P).values(tables[0], rest)
    want, mean, big = attend(q[0], k, v)
    assert ((out[0].cpu().double() - want).abs() <= tolerance(want, mean, big, torch.bfloat16, L)).all()


@gpu
@pytest.mark.parametrize("S", [1, 3, 40])
def test_decode_of_nan_rows_and_of_no_tokens(S):
    """A NaN row makes its own sequence's heads NaN and nothing else; a sequence without tokens is
    NaN; a length past the table counts as the tokens of the table's pages."""
    H, KV, D, P = 8, 2, 128, 16
    lens = [600, 600, 0, 40]
    kv, tables, g = _filled(lens, KV, D, P, torch.bfloat16, 4)
    q = torch.randn(4, H, D, generator=g).bfloat16()
    dev_tab, n = tables.cuda(), torch.tensor([600, 600, 0, 40], dtype=torch.int32).cuda()
    fn = _kv8().paged_decode_attention_kv8
    good = fn(q.cuda(), kv, dev_tab, n, S)
    assert torch.isnan(good[2]).all() and torch.isfinite(good[[0, 1, 3]]).all()
    bad = torch.ones(1, KV, D, dtype=torch.bfloat16, device="cuda")
    bad[0, 1, 7] = math.nan
    at = 451
    page = tables[1, at // P].long().view(1).cuda()
    _kv8().kv8_scatter(bad, bad, kv, page, torch.tensor([at % P]).cuda())
    out = fn(q.cuda(), kv, dev_tab, n, S)
    assert torch.isnan(out[1, H // 2:]).all() and torch.isfinite(out[1, :H // 2]).all()
    assert torch.equal(out[[0, 3]], good[[0, 3]])
    n[0] = 1 << 30
    W = tables.shape[1] * P
    a = fn(q.cuda(), kv, dev_tab, n, S)
    n[0] = W
    assert torch.equal(a[0], fn(q.cuda(), kv, dev_tab, n, S)[0]) or torch.isnan(a[0]).any()


@gpu
def test_decode_over_offsets_past_32_bits():
    """Blocks whose tiles lie past 2^32 bytes of the pool."""
    k8 = _kv8()
    KV, D, P = 8, 128, 16
    NB = (1 << 32) // (KV * P * D) + 40
    kv = k8.kv8_pages(NB, KV, D, P, "cuda")
    L = 300
    blocks = torch.arange(NB - 1, NB - 1 - 19, -1)
    g = torch.Generator().manual_seed(6)
    k, v = (torch.randn(L, KV, D, generator=g).bfloat16() for _ in range(2))
    at = torch.arange(L)
    k8.kv8_scatter(k.cuda(), v.cuda(), kv, blocks[at // P].cuda(), (at % P).cuda())
    pool = Pool(19, KV, D, P)
    pool.put(k, v, at // P, at % P)
    q = torch.randn(1, 32, D, generator=g).bfloat16()
    tab = blocks.int()[None].cuda()
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    ident = torch.arange(19)[None]
    for S in (1, 4):
        out = k8.paged_decode_attention_kv8(q.cuda(), kv, tab, L * one, S)
        _check_rows(out.cpu(), q, pool, ident, [(0, L)], torch.bfloat16)
    out = k8.paged_prefill_attention_kv8(q.cuda(), kv, tab, 0 * one, (L - 1) * one, one, 1)
    _check_rows(out.cpu(), q, pool, ident, [(0, L)], torch.bfloat16)
    gk, gv = k8.kv8_gather(kv, tab, 0 * one, 0 * one, L * one, L, L)
    wk, wv = pool.values(ident[0], range(L))
    assert torch.equal(gk.cpu(), wk.bfloat16()) and torch.equal(gv.cpu(), wv.bfloat16())


@gpu
@pytest.mark.parametrize("S", [1, 6])
def test_decode_buffers_streams_and_graphs(S):
    """Caller-held out and workspace (poisoned first); a strided and an unaligned q; another
    stream; a captured launch replayed over lengths that change between replays."""
    k8 = _kv8()
    H, KV, D, P = 32, 8, 128, 16
    lens = [700, 130]
    kv, tables, g = _filled(lens, KV, D, P, torch.bfloat16, 12)
    tab, n = tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    q = torch.randn(2, H, D, generator=g).bfloat16().cuda()
    want = k8.paged_decode_attention_kv8(q, kv, tab, n, S)
    ws = k8.kv8_workspace(2, H, D, S, "cuda")
    if ws:
        for w in ws:
            w.fill_(math.nan)
    out = torch.full_like(q, math.nan)
    assert k8.paged_decode_attention_kv8(q, kv, tab, n, S, out=out, workspace=ws) is out
    assert torch.equal(out, want)
    wide = torch.zeros(2, D, H, dtype=q.dtype, device="cuda")
    wide.copy_(q.transpose(1, 2))
    odd = torch.zeros(2 * H * D + 1, dtype=q.dtype, device="cuda")[1:].view(2, H, D)
    odd.copy_(q)
    for x in (wide.transpose(1, 2), odd):
        assert torch.equal(k8.paged_decode_attention_kv8(x, kv, tab, n, S), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = k8.paged_decode_attention_kv8(q, kv, tab, n, S)
    s.synchronize()
    assert torch.equal(other, want)
    assert graph_replays_match(
        lambda: k8.paged_decode_attention_kv8(q, kv, tab, n, S, out=out, workspace=ws), lambda: out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k8.paged_decode_attention_kv8(q, kv, tab, n, S, out=out, workspace=ws)
    for a, b in ((1, 130), (333, 17), (700, 1)):
        n.copy_(torch.tensor([a, b], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, k8.paged_decode_attention_kv8(q, kv, tab, n, S))


# ---- GPU: prompt attention -------------------------------------------------------------------

PREFILL = [
    # (H, KV, D, P, [(pos0, nq), ...])
    (4, 4, 64, 16, [(0, 1)]),
    (8, 2, 64, 16, [(0, 16)]),
    (32, 8, 128, 16, [(0, 17)]),
    (32, 8, 128, 16, [(0, 100)]),
    (16, 8, 128, 32, [(37, 5)]),
    (32, 8, 128, 16, [(0, 5), (0, 33), (10, 17), (63, 1)]),
    (64, 8, 128, 16, [(3, 40), (64, 64)]),
    (8, 8, 128, 64, [(100, 70), (0, 2)]),
    (16, 8, 64, 32, [(0, 65), (31, 1)]),
    (20, 5, 64, 16, [(900, 3), (0, 130)]),
    (32, 8, 128, 16, [(1400, 9), (700, 40)]),          # keys divided between workgroups
    (64, 8, 64, 16, [(1000, 30)]),
]


def _prefill_case(H, KV, D, P, segs, dtype, seed, gap=3):
    kv, tables, g = _filled([a + b for a, b in segs], KV, D, P, dtype, seed)
    row0, r = [], gap
    for _, n in segs:
        row0.append(r)
        r += n + gap
    q = (1.5 * torch.randn(r, H, D, generator=g)).to(dtype)
    meta = [torch.tensor(x, dtype=torch.int32) for x in (row0, [a for a, _ in segs], [b for _, b in segs])]
    return kv, tables, q, meta


def _prefill_run(kv, tables, q, meta, out=None):
    return _kv8().paged_prefill_attention_kv8(q.cuda(), kv, tables.cuda(), *(m.cuda() for m in meta),
                                              int(meta[2].max()), out=out)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(PREFILL)))
def test_prefill(case, dtype):
    """Every row of every sequence; the rows between them are left as they were."""
    H, KV, D, P, segs = PREFILL[case]
    kv, tables, q, meta = _prefill_case(H, KV, D, P, segs, dtype, 60 + case)
    out = torch.full(q.shape, 5.0, dtype=dtype, device="cuda")
    _prefill_run(kv, tables, q, meta, out)
    out = out.cpu()
    rows = [(int(meta[0][n]) + j, n, p0 + j + 1) for n, (p0, nq) in enumerate(segs) for j in range(nq)]
    at = [r for r, _, _ in rows]
    _check_rows(out[at], q[at], Pool.of(kv, P), tables, [(n, L) for _, n, L in rows], dtype)
    free = torch.ones(len(q), dtype=torch.bool)
    free[at] = False
    assert (out[free] == 5.0).all()


@gpu
def test_prefill_equals_decode_on_a_long_prompt():
    """5000 rows of one prompt: each within twice the bound of its row of decode attention."""
    H, KV, D, P, L = 8, 2, 128, 16, 5000
    kv, tables, g = _filled([L], KV, D, P, torch.bfloat16, 21)
    q = torch.randn(L, H, D, generator=g).bfloat16()
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    out = _kv8().paged_prefill_attention_kv8(q.cuda(), kv, tables.cuda(), 0 * one, 0 * one, L * one, L)
    pick = torch.tensor([0, 1, 15, 16, 63, 64, 65, 127, 1000, 2047, 2048, 4095, 4990, 4999])
    _check_rows(out[pick.cuda()].cpu(), q[pick], Pool.of(kv, P), tables, [(0, int(i) + 1) for i in pick],
                torch.bfloat16)
    dec = _kv8().paged_decode_attention_kv8(q.cuda(), kv, tables.cuda().expand(L, -1).contiguous(),
                                            torch.arange(1, L + 1, dtype=torch.int32).cuda(), 1)
    # both are within 3 u of the mean of |v|, which is below 4.5 where v has this spread
    assert (out.float() - dec.float()).abs().max() <= 2 * 3 * 2.0 ** -8 * 4.5


@gpu
@pytest.mark.parametrize("pre", [0, 900])
def test_prefill_of_nan_rows(pre):
    """A NaN row of the cache reaches the queries at and behind it, no earlier one and no other
    kv head, also inside the same tile of queries."""
    H, KV, D, P, n, bad = 8, 2, 128, 16, 90, 37
    kv, tables, q, meta = _prefill_case(H, KV, D, P, [(pre, n)], torch.bfloat16, 71, gap=0)
    good = _prefill_run(kv, tables, q, meta)
    row = torch.ones(1, KV, D, dtype=torch.bfloat16, device="cuda")
    row[0, 0, 3] = math.inf
    at = pre + bad
    _kv8().kv8_scatter(row, row, kv, tables[0, at // P].long().view(1).cuda(), torch.tensor([at % P]).cuda())
    out = _prefill_run(kv, tables, q, meta)
    assert torch.equal(out[:bad], good[:bad])
    assert torch.isnan(out[bad:, :H // 2]).all() and torch.isfinite(out[bad:, H // 2:]).all()


@gpu
def test_prefill_metadata_past_its_bounds():
    """Rows past q, past max_nq, past the table's pages, and negative starts are not served; the
    others are those of a correct call, bit for bit."""
    H, KV, D, P = 32, 8, 128, 16
    kv, tables, q, meta = _prefill_case(H, KV, D, P, [(0, 20), (0, 30), (5, 11)], torch.bfloat16, 77)
    good = _prefill_run(kv, tables, q, meta, torch.zeros(q.shape, dtype=q.dtype, device="cuda"))
    fn = _kv8().paged_prefill_attention_kv8
    for i, field, value in ((0, 0, len(q) - 4), (1, 1, tables.shape[1] * P - 7), (2, 2, 1 << 30),
                            (0, 0, -3), (1, 1, -1), (1, 1, (1 << 31) - 5), (2, 2, -4)):
        m = [x.clone() for x in meta]
        m[field][i] = value
        out = torch.zeros(q.shape, dtype=q.dtype, device="cuda")
        fn(q.cuda(), kv, tables.cuda(), *(x.cuda() for x in m), 30, out=out)
        for n in range(3):
            a, b = int(meta[0][n]), int(meta[0][n]) + int(meta[2][n])
            touched = [(int(m[0][k]), int(m[0][k]) + 30) for k in range(3) if k == i]
            if n != i and all(b <= lo or a >= hi for lo, hi in touched):
                assert torch.equal(out[a:b], good[a:b]), (i, field, value, n)


@gpu
@pytest.mark.parametrize("pre", [0, 1500])
def test_a_bound_on_the_rows_may_be_any_number(pre):
    """max_nq far above the rows there are: the same rows, bit for bit, and the same read back."""
    H, KV, D, P = 32, 8, 128, 16
    kv, tables, q, meta = _prefill_case(H, KV, D, P, [(pre, 20), (0, 33)], torch.bfloat16, 78)
    args = (tables.cuda(), *(m.cuda() for m in meta))
    good = _kv8().paged_prefill_attention_kv8(q.cuda(), kv, *args, len(q), out=torch.zeros_like(q).cuda())
    for bound in (len(q) + 1, 1 << 20, (1 << 31) - 1):
        out = torch.zeros_like(q).cuda()
        assert torch.equal(_kv8().paged_prefill_attention_kv8(q.cuda(), kv, *args, bound, out=out), good)
    k0, v0 = _kv8().kv8_gather(kv, *args, 33, len(q))
    k1, v1 = _kv8().kv8_gather(kv, *args, (1 << 31) - 40, len(q))
    rows = torch.cat([torch.arange(int(a), int(a) + int(n)) for a, n in zip(meta[0], meta[2])]).cuda()
    assert torch.equal(k0[rows], k1[rows]) and torch.equal(v0[rows], v1[rows])


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,M,hist,H,KV,D", [(1, 1, 40, 32, 8, 128), (3, 5, 15, 32, 8, 128), (2, 2, 0, 16, 8, 64),
                                             (4, 4, 1500, 32, 8, 128), (2, 20, 300, 8, 8, 128)])
def test_verify_windows(B, M, hist, H, KV, D, dtype):
    """Row (b, j) sees its history and the window up to itself."""
    P = 16
    lens = [hist + b + M for b in range(B)]
    kv, tables, g = _filled(lens, KV, D, P, dtype, 90 + M)
    q = (1.5 * torch.randn(B, M, H, D, generator=g)).to(dtype)
    out = _kv8().paged_verify_attention_kv8(q.cuda(), kv, tables.cuda(),
                                            torch.tensor(lens, dtype=torch.int32).cuda())
    seen = [(b, lens[b] - (M - 1 - j)) for b in range(B) for j in range(M)]
    _check_rows(out.cpu().view(-1, H, D), q.view(-1, H, D), Pool.of(kv, P), tables, seen, dtype)


@gpu
def test_verify_windows_that_see_no_token():
    """A window longer than its sequence: rows before the first token are NaN, the others as usual;
    a sequence without tokens is NaN."""
    H, KV, D, P, M = 8, 2, 128, 16, 4
    kv, tables, g = _filled([2, 50, 0], KV, D, P, torch.bfloat16, 5)
    q = torch.randn(3, M, H, D, generator=g).bfloat16()
    lens = torch.tensor([2, 50, 0], dtype=torch.int32).cuda()
    out = _kv8().paged_verify_attention_kv8(q.cuda(), kv, tables.cuda(), lens).cpu()
    assert torch.isnan(out[0, :2]).all() and torch.isnan(out[2]).all()
    rows = torch.stack([out[0, 2], out[0, 3], out[1, 0], out[1, 3]])
    qs = torch.stack([q[0, 2], q[0, 3], q[1, 0], q[1, 3]])
    _check_rows(rows, qs, Pool.of(kv, P), tables, [(0, 1), (0, 2), (1, 47), (1, 50)], torch.bfloat16)


# ---- GPU: refusals and empty calls -----------------------------------------------------------


@gpu
def test_refusals():
    k8 = _kv8()
    kv = k8.kv8_pages(4, 2, 128, 16, "cuda")
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16, device="cuda")
    tab = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    row = torch.zeros(1, 2, 128, dtype=torch.bfloat16, device="cuda")
    i64 = torch.zeros(1, dtype=torch.int64, device="cuda")
    dec = k8.paged_decode_attention_kv8
    for call in (
            lambda: dec(q[..., :64], kv, tab, one),                               # head size
            lambda: dec(q[:, :3], kv, tab, one),                                  # heads
            lambda: dec(q, kv, tab.long(), one),                                  # table type
            lambda: dec(q, kv, tab[:, :0], one),                                  # no pages
            lambda: dec(q, kv, tab, one.expand(2)),                               # lengths
            lambda: dec(q, kv, tab, one, 0),                                      # splits
            lambda: dec(q, kv, tab, one, out=q.float()),                          # out type
            lambda: dec(q, kv, tab, one, 3, workspace=(one.float(), one.float())),
            lambda: dec(q, k8.KV8Pages(kv.k, kv.v[:3], kv.scales), tab, one),
            lambda: dec(q, k8.KV8Pages(kv.k.int(), kv.v, kv.scales), tab, one),
            lambda: dec(q, k8.KV8Pages(kv.k, kv.v, kv.scales[..., :16]), tab, one),
            lambda: k8.kv8_scatter(row, row[:, :1], kv, i64, i64),
            lambda: k8.kv8_scatter(row, row.float(), kv, i64, i64),
            lambda: k8.kv8_scatter(row, row, kv, one, i64),
            lambda: k8.kv8_scatter(row, row, kv, i64.expand(2), i64),
            lambda: k8.kv8_gather(kv, tab, one, one, one.expand(2), 1, 1),
            lambda: k8.kv8_gather(kv, tab, one, one, one, 1, -1),
            lambda: k8.paged_prefill_attention_kv8(q, kv, tab, one, one, one.long(), 1),
            lambda: k8.paged_verify_attention_kv8(q[None, :, :, :64], kv, tab, one),
            lambda: k8.qkv_norm_rope_kv8(row.view(1, -1), kv, i64, i64, i64, torch.ones(64, device="cuda"),
                                         row[0, 0], row[0, 0], 1e-6, 4)):
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(NotImplementedError):
        dec(q.float(), kv, tab, one)
    with pytest.raises(NotImplementedError):
        dec(q.expand(1, 4, 128).repeat(1, 8, 1), kv, tab, one)
    with pytest.raises(ValueError):
        k8.kv8_scatter(row.double(), row.double(), kv, i64, i64)
    with pytest.raises(ValueError):
        k8.kv8_gather(kv, tab, one, one, one, 1, 1, dtype=torch.float64)
    assert not kv.scales.any()


@gpu
def test_empty_calls():
    k8 = _kv8()
    kv = k8.kv8_pages(2, 2, 128, 16, "cuda")
    none = torch.zeros(0, 2, 128, dtype=torch.bfloat16, device="cuda")
    i32 = torch.zeros(0, dtype=torch.int32, device="cuda")
    i64 = torch.zeros(0, dtype=torch.int64, device="cuda")
    tab = torch.zeros(0, 0, dtype=torch.int32, device="cuda")
    k8.kv8_scatter(none, none, kv, i64, i64)
    assert k8.kv8_gather(kv, tab, i32, i32, i32, 0, 0)[0].shape == (0, 2, 128)
    assert k8.paged_decode_attention_kv8(none, kv, tab, i32).shape == none.shape
    assert k8.paged_prefill_attention_kv8(none, kv, tab, i32, i32, i32, 0).shape == none.shape
    assert k8.paged_verify_attention_kv8(none[:, None], kv, tab, i32).shape == (0, 1, 2, 128)
    assert k8.paged_verify_attention_kv8(none[:, None].expand(0, 3, 2, 128), kv, tab, i32).shape == (0, 3, 2, 128)
    w = torch.ones(128, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(0, 6 * 128, dtype=torch.bfloat16, device="cuda")
    assert k8.qkv_norm_rope_kv8(x, kv, i64, i64, i64, torch.ones(64, device="cuda"), w, w, 1e-6, 2).shape == none.shape
    torch.cuda.synchronize()
