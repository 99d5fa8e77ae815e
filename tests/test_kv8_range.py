"""The ends of the 8-bit cache's range: numbers near the largest of their type are held as the
largest that stays finite when read, so V is finite whatever was written and a row reaches only
the queries that see it."""
import math

import numpy as np
import pytest
import torch

from oracle.kv8_ref import E4M3, Pool, attend, quantise_row, tolerance

TOP = math.ldexp(240.0, 120)             # the largest number of the grid below 2^128


def _kv8():
    from acorninfer_amd.ops import kv8
    return kv8


@pytest.mark.parametrize("x,held", [(TOP, TOP), (247.9 * 2.0 ** 120, TOP), (248 * 2.0 ** 120, TOP),
                                    (float(torch.finfo(torch.bfloat16).max), TOP),
                                    (-float(torch.finfo(torch.float32).max), -TOP),
                                    (231.0 * 2.0 ** 120, 224 * 2.0 ** 120), (447.9 * 2.0 ** 119, 448 * 2.0 ** 119)])
def test_oracle_holds_the_largest_numbers_as_finite_ones(x, held):
    b, code, ok = quantise_row(np.array([x, 1.0]), False)
    assert ok and E4M3[b[0]] * 2.0 ** (code - 127) == held
    assert np.isfinite(np.float32(held))
    assert torch.isfinite(torch.tensor(held, dtype=torch.float64).to(torch.bfloat16))


def _huge(dtype, n, KV, D, seed):
    """Rows with numbers around and above the border, at any place, beside ordinary ones."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, KV, D, generator=g)
    top = torch.finfo(dtype).max
    big = torch.tensor([top, -top, 0.97 * top, 0.9688 * top, -0.94 * top, 0.9 * top, 0.6 * top])
    big = torch.cat([big.clamp(-top, top), torch.tensor([min(TOP, top), -min(TOP, top), min(248 * 2.0 ** 120, top)])])
    for i in range(n):
        for h in range(KV):
            if (i + h) % 3:
                x[i, h, (7 * i + 3 * h) % D] = big[(i + h) % len(big)]
    return x.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_scatter_and_gather_at_the_ends_of_a_type(dtype):
    """The oracle's bytes, and finite rows read back."""
    R, KV, D, P = 40, 3, 128, 16
    k, v = _huge(dtype, R, KV, D, 1), _huge(dtype, R, KV, D, 2)
    assert torch.isfinite(k).all() and torch.isfinite(v).all()
    at = torch.arange(R)
    pool = Pool(3, KV, D, P)
    pool.put(k, v, at // P, at % P, dtype == torch.float16)
    kv = _kv8().kv8_pages(3, KV, D, P, "cuda")
    _kv8().kv8_scatter(k.cuda(), v.cuda(), kv, (at // P).cuda(), (at % P).cuda())
    for a, b in zip(kv, (pool.k, pool.v, pool.scales)):
        assert np.array_equal(a.cpu().numpy(), b)
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    tab = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    for x, want in zip(_kv8().kv8_gather(kv, tab, 0 * one, 0 * one, R * one, R, R, dtype=dtype),
                       pool.values(range(3), range(R))):
        assert torch.isfinite(x).all() and torch.equal(x.cpu(), want.to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("planes", [0, 2])
def test_qkv_epilogue_at_the_ends_of_32_bits(dtype, planes):
    """v of a projection that reaches the largest numbers of its type: the oracle's bytes."""
    R, H, KV, D, P = 33, 4, 2, 64, 16
    src = torch.float32 if planes else dtype
    v = _huge(src, R, KV, D, 3).view(R, KV * D)
    g = torch.Generator().manual_seed(4)
    x = torch.cat([torch.randn(R, (H + KV) * D, generator=g).to(src), v], 1)
    qkv = torch.stack([x, torch.zeros_like(x)]) if planes else x
    kv = _kv8().kv8_pages(3, KV, D, P, "cuda")
    at = torch.arange(R)
    w = torch.ones(D, dtype=dtype, device="cuda")
    _kv8().qkv_norm_rope_kv8(qkv.cuda(), kv, (at // P).cuda(), (at % P).cuda(), at.cuda(),
                             torch.ones(D // 2, device="cuda"), w, w, 1e-6, H)
    pool = Pool(3, KV, D, P)
    pool.put(v.view(R, KV, D), v.view(R, KV, D), at // P, at % P, dtype == torch.float16)
    held = Pool.of(kv, P)
    assert np.array_equal(held.v, pool.v) and np.array_equal(held.scales[..., 16:], pool.scales[..., 16:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("pre", [0, 900])
def test_a_row_of_the_largest_numbers_reaches_no_earlier_query(dtype, where, pre):
    """In v: queries before such a row, in its own tile too, keep their bits. (Those behind it hold
    its multiple by a weight that may pass 1 before the sum divides it: finite in fp16, whose 61440
    is far from the sums' 2^128.) In k: they stay within their bound, as a greater score of a later
    query moves the running maxima of the queries beside it, and with them the roundings."""
    H, KV, D, P, n, bad = 8, 2, 128, 16, 90, 37
    L = pre + n
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(L, KV, D, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(n, H, D, generator=g).to(dtype).cuda()
    at = torch.arange(L)
    NB = -(-L // P)
    meta = [torch.tensor([x], dtype=torch.int32).cuda() for x in (0, pre, n)]
    tab = torch.arange(NB, dtype=torch.int32, device="cuda")[None]
    outs = []
    for plant in (False, True):
        kv = _kv8().kv8_pages(NB, KV, D, P, "cuda")
        if plant:
            (k if where == "k" else v)[pre + bad, :, 5] = torch.finfo(dtype).max
        _kv8().kv8_scatter(k.cuda(), v.cuda(), kv, (at // P).cuda(), (at % P).cuda())
        outs.append(_kv8().paged_prefill_attention_kv8(q, kv, tab, *meta, n))
        win = _kv8().paged_verify_attention_kv8(q[None], kv, tab, torch.tensor([L], dtype=torch.int32).cuda())
        outs.append(win[0])
    for good, out in ((outs[0], outs[2]), (outs[1], outs[3])):
        assert torch.isfinite(good).all()
        if where == "v":
            assert torch.equal(out[:bad], good[:bad])
        else:
            hk, hv = Pool.of(kv, P).values(range(NB), range(pre + bad))
            for i in range(bad):
                want, mean, big = attend(q[i].cpu(), hk[:pre + i + 1], hv[:pre + i + 1])
                assert ((out[i].cpu().double() - want).abs() <= tolerance(want, mean, big, dtype, pre + i)).all()
        if where == "v" and dtype == torch.float16:
            assert torch.isfinite(out).all()
