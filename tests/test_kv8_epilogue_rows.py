"""The qkv epilogue of the 8-bit cache at 1024 rows and around: a workgroup takes all heads of its
token in several passes, the next pass's heads requested ahead, and runs of 128 tokens are dealt out
by 16. Fewer rows: test_kv8.py."""
import numpy as np
import pytest
import torch

from oracle.kv8_ref import E4M3, Pool, quantise_row

gpu = pytest.mark.gpu


def _kv8():
    from acorninfer_amd.ops import kv8
    return kv8


def _borders(R):
    """Rows at the borders of runs of 128 tokens and of 16, the ends, and some between."""
    rows = {0, 1, 15, 16, 17, 127, 128, 129, 143, 144, 255, 256, 511, 512, 895, 896, 1000, 1023, 1024,
            R - 129, R - 128, R - 17, R - 16, R - 2, R - 1} | set(range(R // 128 * 128 - 1, R, 9))
    return torch.tensor(sorted(r for r in rows if 0 <= r < R))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,KV,D,P,R,S", [(32, 8, 128, 16, 1157, 0), (20, 5, 64, 16, 1157, 2), (64, 8, 128, 32, 1029, 0),
                                          (20, 5, 128, 16, 1024, 0), (8, 8, 64, 16, 1279, 2), (1, 1, 64, 16, 1100, 0),
                                          (32, 8, 64, 16, 1023, 0)])
def test_qkv_epilogue_of_many_rows(H, KV, D, P, R, S, dtype):
    """q of every row within its roundings; k and v of the rows at the borders within a rounding to
    e4m3, of all rows within a step of it; slots that no row names as they were."""
    g = torch.Generator().manual_seed(R + H)
    width = (H + 2 * KV) * D
    x = torch.randn(*((S, R, width) if S else (R, width)), generator=g) * 0.7
    x = x if S else x.to(dtype)
    pos = torch.randint(0, 131072, (R,), generator=g)
    inv_freq = 1.0 / 1e6 ** (torch.arange(0, D, 2).float() / D)
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(dtype) for _ in range(2))
    pool = Pool(R // P + 3, KV, D, P)
    kv = _kv8().kv8_pages(pool.NB, KV, D, P, "cuda")
    at = torch.randperm(pool.NB * P, generator=g)[:R]
    q = _kv8().qkv_norm_rope_kv8(x.cuda(), kv, (at // P).cuda(), (at % P).cuda(), pos.cuda(), inv_freq.cuda(),
                                 qw.cuda(), kw.cuda(), 1e-6, H).cpu()
    y = x.double()
    mag = (y.abs().sum(0) if S else y.abs()).view(R, H + 2 * KV, D)
    y = (y.sum(0) if S else y).view(R, H + 2 * KV, D)
    w = torch.cat([qw.double().expand(H, D), kw.double().expand(KV, D)])
    inv = 1 / (y[:, :H + KV].square().mean(-1, keepdim=True) + 1e-6).sqrt()
    z, mag_z = y[:, :H + KV] * inv * w, mag[:, :H + KV] * inv * w.abs()
    ang = pos.double()[:, None, None] * inv_freq.double()
    a, b = z.chunk(2, -1)
    rot = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)
    # 32-bit steps: the planes, the mean square, the root, two products, cos and sin, the sum:
    # under 64 of 2^-24 of the magnitudes
    ma, mb = mag_z.chunk(2, -1)
    eps = 64 * 2.0 ** -24 * torch.cat([ma + mb, ma + mb], -1)
    u = torch.finfo(dtype).eps / 2
    assert ((q.double() - rot[:, :H]).abs() <= u * (rot[:, :H].abs() + eps[:, :H]) + eps[:, :H] + 2.0 ** -25).all()
    held = Pool.of(kv, P)
    got_k, got_v = held.values(np.arange(pool.NB), at)
    pick = _borders(R)
    for got, want, e in ((got_k, rot[:, H:], eps[:, H:]), (got_v, y[:, H + KV:], 64 * 2.0 ** -24 * mag[:, H + KV:])):
        top = (want.abs() + e).amax(-1, keepdim=True)
        grid = 2.0 ** (torch.floor(torch.log2(top)) - 7)               # 2^e at most
        assert ((got - want).abs() <= 2.0 ** -4 * (want.abs() + e) + 2.0 ** -10 * grid + e).all()
        same = []
        for row, have in zip(want[pick].reshape(-1, D).numpy(), got[pick].reshape(-1, D).numpy()):
            byte, code, _ = quantise_row(row, dtype == torch.float16)
            same.append((E4M3[byte] * 2.0 ** (code - 127) == have).mean())
        # (bytes differ only where 64 and 32 bits fall on two sides of a border)
        assert np.mean(same) > 0.999
    keep = torch.ones(pool.NB * P, dtype=torch.bool)
    keep[at] = False
    rest = torch.arange(pool.NB * P)[keep]
    assert len(rest) == pool.NB * P - R and all((t == 0).all() for t in held.values(np.arange(pool.NB), rest))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_rows_equal_few(dtype):
    """The same rows in one call and in calls of 100: the same q and the same bytes (each row's
    arithmetic does not depend on the form)."""
    H, KV, D, P, R = 32, 8, 128, 16, 1157
    g = torch.Generator().manual_seed(2)
    x = torch.randn(R, (H + 2 * KV) * D, generator=g).to(dtype).cuda()
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(dtype).cuda()
    inv_freq = (1.0 / 1e6 ** (torch.arange(0, D, 2).float() / D)).cuda()
    at = torch.arange(R, device="cuda")
    kvs = [_kv8().kv8_pages(R // P + 1, KV, D, P, "cuda") for _ in range(2)]
    one = _kv8().qkv_norm_rope_kv8(x, kvs[0], at // P, at % P, 7 * at, inv_freq, w, w, 1e-6, H)
    few = torch.cat([_kv8().qkv_norm_rope_kv8(x[i:i + 100], kvs[1], at[i:i + 100] // P, at[i:i + 100] % P,
                                              7 * at[i:i + 100], inv_freq, w, w, 1e-6, H)
                     for i in range(0, R, 100)])
    assert torch.equal(one, few)
    assert all(torch.equal(a, b) for a, b in zip(*kvs))
