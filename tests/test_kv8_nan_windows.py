"""NaN rows of the 8-bit cache under verify windows, whose V is bf16 in either type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,hist", [(5, 40), (5, 1500), (40, 30), (40, 1500)])
def test_a_nan_row_reaches_the_window_rows_that_see_it(m, hist, dtype):
    """One kv head of a drafted token holds an infinity: the window's rows from it on are NaN in that
    head's q heads, all others keep their bits; bytes behind the sequence may be anything."""
    from acorninfer_amd.ops import kv8
    H, KV, D, P = 8, 2, 128, 16
    L = hist + m
    NB = -(-L // P)
    g = torch.Generator().manual_seed(m + hist)
    k, v = (torch.randn(L, KV, D, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(1, m, H, D, generator=g).to(dtype).cuda()
    kv = kv8.KV8Pages(*(torch.full((NB, KV, 1, n), 255, dtype=torch.uint8, device="cuda")
                        for n in (16 * D, 16 * D, 32)))
    at = torch.arange(L)
    tab = torch.arange(NB, dtype=torch.int32, device="cuda")[None]
    lens = torch.full((1,), L, dtype=torch.int32, device="cuda")
    outs = []
    for bad in (None, hist + m // 2):
        if bad is not None:
            v[bad, 0, 3] = math.inf
        kv8.kv8_scatter(k.cuda(), v.cuda(), kv, (at // P).cuda(), (at % P).cuda())
        outs.append(kv8.paged_verify_attention_kv8(q, kv, tab, lens)[0])
    good, out = outs
    first = m // 2
    assert torch.isfinite(good).all()
    assert torch.equal(out[:first], good[:first]) and torch.equal(out[:, H // 2:], good[:, H // 2:])
    assert torch.isnan(out[first:, :H // 2]).all()
