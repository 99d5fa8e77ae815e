"""How near attention over the 8-bit cache is to 64 bits: decode and verify windows
take the probabilities in two bf16 terms, so that only the result's own rounding counts; they and
prompt rows keep the weight of many tokens far below one (an attention sink)."""
import pytest
import torch

from oracle.kv8_ref import Pool, attend, tolerance

gpu = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
P = 16


def _kv8():
    from acorninfer_amd.ops import kv8
    return kv8


def _cache(k, v):
    """k, v [L, KV, D] as tokens 0 .. L - 1 of pages in order."""
    L, KV, D = k.shape
    NB = -(-L // P)
    kv = _kv8().kv8_pages(NB, KV, D, P, "cuda")
    at = torch.arange(L)
    _kv8().kv8_scatter(k.cuda(), v.cuda(), kv, (at // P).cuda(), (at % P).cuda())
    return kv, torch.arange(NB, dtype=torch.int32, device="cuda")[None]


def _run(form, q, kv, tab, L):
    """q [H, D] as the last token of a sequence of L: by decode in n splits, as the last row of a
    window of n, or as the last of n prompt rows."""
    kind, n = form
    lens = torch.full((1,), L, dtype=torch.int32, device="cuda")
    if kind == "decode":
        return _kv8().paged_decode_attention_kv8(q[None].cuda(), kv, tab, lens, n)[0].cpu()
    if kind == "window":
        return _kv8().paged_verify_attention_kv8(q.expand(1, n, *q.shape).cuda(), kv, tab, lens)[0, -1].cpu()
    one = torch.ones_like(lens)
    return _kv8().paged_prefill_attention_kv8(q.expand(n, *q.shape).cuda(), kv, tab, 0 * one, lens - n, n * one,
                                              n)[-1].cpu()


def _close(heads, D, dtype, L):
    """Half the tokens have a score delta below the others' and values of the other sign: the result
    is tanh(delta / 2), and 0 where p = 1 - delta is rounded to 1 (delta below half a step of the
    type)."""
    part = torch.linspace(0.6, 0.95, heads, dtype=torch.float64)
    delta = part * (2.0 ** -9 if dtype == torch.bfloat16 else 2.0 ** -12)
    q = torch.zeros(heads, D)
    q[:, 0] = -delta * D ** 0.5
    k = torch.zeros(L, 1, D)
    k[1::2, 0, 0] = 1.0
    v = torch.ones(L, 1, D)
    v[1::2] = -1.0
    return q.to(dtype), k.to(dtype), v.to(dtype)


def test_the_bound_tells_one_term_from_two():
    """CPU: the weights rounded once to either type miss the bound of two terms on these inputs."""
    for dtype in DTYPES:
        q, k, v = _close(8, 64, dtype, 600)
        want, mean, big = attend(q, k.double(), v.double())
        tol = tolerance(want, mean, big, dtype, 600, terms=2)
        s = (q.double() @ k[:, 0].double().T) * 64 ** -0.5
        p = torch.exp(s)
        one = p.to(dtype).double()
        hi = (p.float().view(torch.int32) & -65536).view(torch.float32)
        two = hi.double() + (p.float() - hi).bfloat16().double()

        def out(w, l):
            return (w @ v[:, 0].double() / l.sum(-1, keepdim=True)).to(dtype).double()
        assert ((out(one, one) - want).abs() > tol).all()
        assert ((out(two, p) - want).abs() <= tol).all() and ((out(two, two) - want).abs() <= tol).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,heads,L", [(128, 4, 600), (64, 8, 600), (128, 1, 3000), (128, 8, 34)])
@pytest.mark.parametrize("form", [("decode", 1), ("decode", 3), ("decode", 64), ("window", 2), ("window", 40)])
def test_two_terms(form, D, heads, L, dtype):
    if form[0] == "window":
        L = max(L, 80)
    q, k, v = _close(heads, D, dtype, L)
    out = _run(form, q, *_cache(k, v), L)
    want, mean, big = attend(q, k.double(), v.double())
    tol = tolerance(want, mean, big, dtype, L, terms=2)
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"{float((err / tol).max()):.2f} of the bound"


def _random(B, L, H, KV, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    k = (torch.randn(L, KV, D, generator=g) * torch.exp(0.5 * torch.randn(1, 1, D, generator=g))).to(dtype)
    v = torch.randn(L, KV, D, generator=g).to(dtype)
    return torch.randn(B, H, D, generator=g).to(dtype), k, v


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,L", [(32, 40), (16, 400), (8, 1600)])
def test_decode_and_window_rows_are_off_by_the_results_rounding(H, L, dtype):
    """Rows through decode and through windows of five, against 64 bits: the error is that of
    rounding the result to its type, within a percent (20000 outputs and more: the norms are known
    to within one; what 32 bits and two terms add is below a hundredth of a rounding)."""
    KV, D, m, B = 8, 128, 5, 160
    q, k, v = _random(B, L, H, KV, D, dtype, L)
    kv, tab = _cache(k, v)
    pool = Pool.of(kv, P)
    held = pool.values(range(pool.NB), range(L))
    seen = [L - (m - 1 - i % m) for i in range(B)]
    exact = torch.stack([attend(x, held[0][:n], held[1][:n])[0] for x, n in zip(q, seen)])
    lens = torch.tensor(seen, dtype=torch.int32, device="cuda")
    rows = _kv8().paged_decode_attention_kv8(q.cuda(), kv, tab.expand(B, -1).contiguous(), lens).cpu()
    wins = _kv8().paged_verify_attention_kv8(q.view(B // m, m, H, D).cuda(), kv,
                                             tab.expand(B // m, -1).contiguous(),
                                             torch.full((B // m,), L, dtype=torch.int32, device="cuda"))
    best = float((exact.to(dtype).double() - exact).norm())
    for name, x in (("decode", rows), ("windows", wins.view(B, H, D).cpu())):
        assert float((x.double() - exact).norm()) <= 1.01 * best, name


PROMPT_STEP = 2.0 ** -25 * 2.0 ** -7       # half of fp16's least step, of weights held times 2^7
SINK_GAPS = (10.0, 16.5, 17.0, 17.5, 20.0, 22.0)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", [("decode", 1), ("decode", 16), ("window", 3), ("window", 40),
                                  ("prompt", 1), ("prompt", 70)])
@pytest.mark.parametrize("at", [0, 2000])
def test_many_tokens_far_below_one_keep_their_weight(at, form, dtype):
    """One token whose score is `gap` above that of 4000 others, and whose values are 0: the result
    is the others' weight, exp(-gap) each."""
    L, D, KV = 4001, 128, 1
    g = torch.Generator().manual_seed(3)
    k = torch.zeros(L, KV, D)
    k[at, 0, 0] = 1.0
    v = 1000.0 * (1.0 + torch.rand(L, KV, D, generator=g))
    v[at] = 0.0
    kv, tab = _cache(k.to(dtype), v.to(dtype))
    pool = Pool.of(kv, P)
    hk, hv = pool.values(range(pool.NB), range(L))
    for first in range(0, len(SINK_GAPS), 2):
        q = torch.zeros(2, D)
        q[:, 0] = torch.tensor(SINK_GAPS[first:first + 2]) * D ** 0.5
        q = q.to(dtype)
        out = _run(form, q, kv, tab, L).double()
        want, mean, big = attend(q, hk, hv)
        tol = tolerance(want, mean, big, dtype, L, terms=1 if form[0] == "prompt" else 2)
        if form[0] == "prompt" and dtype == torch.float16:
            tol = tol + PROMPT_STEP * hv.abs().sum(0)          # (each weight, of a sum above 1)
        err = (out - want).abs()
        assert (err <= tol).all(), (SINK_GAPS[first], float((err / tol).max()), float((out / want).mean()))


@gpu
@pytest.mark.parametrize("order", ["rising", "falling"])
def test_prompt_weights_stay_within_fp16(order):
    """Scores that rise or fall by less than the maximum's slack from step to step: the largest
    weights are 2^15, and no sum of them is lost."""
    L, D, KV, H = 700, 64, 1, 8
    g = torch.Generator().manual_seed(5)
    k = torch.zeros(L, KV, D)
    k[:, 0, 0] = torch.linspace(0, 448, L) if order == "rising" else torch.linspace(448, 0, L)
    v = torch.randn(L, KV, D, generator=g)
    kv, tab = _cache(k.half(), v.half())
    pool = Pool.of(kv, P)
    hk, hv = pool.values(range(pool.NB), range(L))
    q = torch.zeros(H, D)
    q[:, 0] = torch.linspace(0.02, 2.0, H)
    q = q.half()
    out = _run(("prompt", 1), q, kv, tab, L).double()
    want, mean, big = attend(q, hk, hv)
    err = (out - want).abs()
    tol = tolerance(want, mean, big, torch.float16, L)
    assert (err <= tol).all(), float((err / tol).max())
