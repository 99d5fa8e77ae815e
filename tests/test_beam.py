"""Beam search's operators (ops/beam.py) against oracle/beam_ref.py: selection in 64 bits,
bookkeeping, the cache that follows the beams, hypotheses out of the logs. Whole numbers are
exact. A selected score is off by its rounding to fp32 and by the error of the row's sum:
`score_bound`."""
import itertools
import math

import pytest
import torch

from gpu_utils import graph_replays_match
from oracle import beam_ref as ref

gpu = pytest.mark.gpu
INF = math.inf
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _beam():
    from acorninfer_amd.ops import beam
    return beam


def score_bound(want: torch.Tensor, vocab: int) -> torch.Tensor:
    """s = score + x - lse is rounded once, from 64 bits (2^-24 |s|). lse is off by the relative error
    of the sum of exponentials: each is 2^-22 or better for the largest (the exponent's argument t
    log2 e is off by 2^-23 |t|, weighted with e^t: |t| e^t < 1), and a lane adds at most
    vocab / 256 + 32 of them one by one, then 6 across lanes and 3 across waves, 2^-24 each."""
    return 2.0 ** -24 * (want.abs() + vocab / 256 + 32 + 9 + 8)


# ---- CPU: the oracle and the refusals ---------------------------------------------------------


def test_search_of_the_oracle_with_room_for_all_is_exhaustive():
    """With as many beams as there are prefixes nothing is dropped: the best hypothesis is the best of
    all token rows that end with the end token or are full."""
    V, T, end = 3, 3, 0
    g = torch.Generator().manual_seed(5)
    table = {}

    def logits_of(toks):
        return table.setdefault(toks, torch.randn(V, generator=g))

    def score(row):
        return sum(float(torch.log_softmax(logits_of(row[:i]).double(), -1)[t])
                   for i, t in enumerate(row))

    every = []
    for n in range(1, T + 1):
        for row in itertools.product(range(V), repeat=n):
            if end in row[:-1] or (row[-1] != end and n < T):
                continue
            every.append((score(row) / n ** 0.7, row))
    want = sorted(every, key=lambda h: -h[0])
    got = ref.search_ref(logits_of, 9, T, {end}, alpha=0.7)
    assert [h[1] for h in got[:3]] == [h[1] for h in want[:3]]
    assert abs(got[0][0] - want[0][0]) < 1e-12


@pytest.mark.parametrize("W", [1, 2, 3, 5, 32])
def test_pages_of_the_oracle_stay_apart(W):
    """Whatever the parents: W different pages, each with its parent's tokens, copies out of pages
    that nothing is copied into."""
    g = torch.Generator().manual_seed(W)
    for _ in range(50):
        par = torch.randint(0, W, (W,), generator=g).tolist()
        page = torch.randperm(2 * W, generator=g)[:W].tolist()
        taken, copies = ref.deal_pages(par, page)
        assert sorted(taken) == sorted(page)
        held = {p: p for p in page}
        for src, dst in copies:
            held[dst] = held[src]
        assert [held[t] for t in taken] == [page[p] for p in par]
        assert not {s for s, _ in copies} & {d for _, d in copies}


def _cpu_state(G=2, W=3, T=4):
    return _beam().beam_state(G, W, T, "cpu")


def test_a_new_state():
    st = _cpu_state()
    assert st.scores.tolist() == [[0.0, -INF, -INF]] * 2
    assert st.fin_scores.tolist() == [[-INF] * 3] * 2 and int(st.fin_length.sum()) == 0
    buf = torch.zeros(6, dtype=torch.int64)
    assert _beam().beam_state(2, 3, 4, "cpu", ids=buf).ids.data_ptr() == buf.data_ptr()
    with pytest.raises(NotImplementedError):
        _beam().beam_state(1, 33, 4, "cpu")


def test_select_refusals():
    b = _beam()
    x, s = torch.zeros(6, 10), torch.zeros(2, 3)
    for bad in (lambda: b.beam_select(x[:5], s, 4), lambda: b.beam_select(x, s.double(), 4),
                lambda: b.beam_select(x, s, 0), lambda: b.beam_select(x, s, 31),
                lambda: b.beam_select(x, s.t(), 4), lambda: b.beam_select(x.view(2, 3, 10), s, 4),
                lambda: b.beam_select(x[:, :0], s, 1), lambda: b.beam_select(x, s[:, :0], 1),
                lambda: b.beam_select(x, s, 4, out=b.BeamCandidates(s, s, s, s))):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(NotImplementedError):
        b.beam_select(torch.zeros(6, 100), s, 65)
    with pytest.raises(NotImplementedError):
        b.beam_select(torch.zeros(33, 100), torch.zeros(1, 33), 4)
    with pytest.raises(ValueError):
        b.beam_select(x.double(), s, 4)
    with pytest.raises(ValueError):                         # right, but not on a GPU
        b.beam_select(x, s, 4)


def test_advance_refusals():
    b = _beam()
    st = _cpu_state()
    i32, i64 = torch.int32, torch.int64
    cand = b.BeamCandidates(torch.zeros(2, 6), torch.zeros(2, 6, dtype=i32), torch.zeros(2, 6, dtype=i64))
    ends = torch.tensor([1])
    for bad in (lambda: b.beam_advance(st._replace(length=st.length.long()), cand, ends),
                lambda: b.beam_advance(st._replace(parents=st.parents[:1]), cand, ends),
                lambda: b.beam_advance(st._replace(token_log=st.token_log[:2]), cand, ends),
                lambda: b.beam_advance(st, cand._replace(beam=cand.token), ends),
                lambda: b.beam_advance(st, cand._replace(score=cand.score[:1]), ends),
                lambda: b.beam_advance(st, cand, ends.int()),
                lambda: b.beam_advance(st, cand, ends[None]),
                lambda: b.beam_advance(st, cand, ends, out=_cpu_state())):       # other logs
        with pytest.raises(AssertionError):
            bad()
    for alpha in (math.nan, INF):
        with pytest.raises(ValueError):
            b.beam_advance(st, cand, ends, length_penalty=alpha)
    wide = [torch.zeros(2, 65, dtype=t.dtype) for t in cand[:3]]
    with pytest.raises(NotImplementedError):
        b.beam_advance(st, b.BeamCandidates(*wide), ends)
    with pytest.raises(ValueError):
        b.beam_advance(st, cand, ends)


def test_reorder_and_trace_refusals():
    b = _beam()
    pool = torch.zeros(2, 4, 16, 2, 8, dtype=torch.bfloat16)
    i32 = torch.int32
    tab, lens, par = torch.zeros(4, 3, dtype=i32), torch.zeros(2, 2, dtype=i32), torch.zeros(2, 2, dtype=i32)
    tiles, codes = torch.zeros(2, 4, 2, 1, 1024, dtype=torch.uint8), torch.zeros(2, 4, 2, 1, 32, dtype=torch.uint8)
    for bad in (lambda: b.beam_reorder(pool, pool[:1], tab, lens, par),
                lambda: b.beam_reorder(pool, pool, tab[:3], lens, par),
                lambda: b.beam_reorder(pool, pool, tab.long(), lens, par),
                lambda: b.beam_reorder(pool, pool, tab, lens[:1], par),
                lambda: b.beam_reorder(pool, pool, tab, lens, par.long()),
                lambda: b.beam_reorder(pool[0], pool[0], tab, lens, par),
                lambda: b.beam_reorder(pool.int(), pool.int(), tab, lens, par),
                lambda: b.beam_reorder(pool.transpose(2, 3), pool.transpose(2, 3), tab, lens, par),
                lambda: b.beam_reorder(tiles, tiles, tab, lens, par, scale_pool=codes[:1]),
                lambda: b.beam_reorder(pool, pool, tab, lens, par, scale_pool=codes)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(ValueError):
        b.beam_reorder(pool, pool, tab, lens, par)
    log = torch.zeros(5, 2, 3, dtype=i32)
    st = torch.zeros(2, 4, dtype=i32)
    for bad in (lambda: b.beam_trace(log, log[:4], st, st), lambda: b.beam_trace(log.long(), log, st, st),
                lambda: b.beam_trace(log, log, st[:1], st), lambda: b.beam_trace(log, log, st, st.long()),
                lambda: b.beam_trace(log, log, st, st, out=torch.zeros(2, 4, 5))):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(ValueError):
        b.beam_trace(log, log, st, st)


def test_entries_refuse_without_a_gpu():
    from acorninfer_amd import _lib
    L, p = _lib.lib(), 64                                   # a pointer that is never followed
    def select(G=1, W=2, V=10, k=4, dtype=2, x=p, ws=p, ws_bytes=1 << 20, stride=10):
        return L.acorn_beam_select(x, stride, p, G, W, V, k, p, p, p, p, ws, ws_bytes, dtype, None)
    assert select(W=0) == select(V=0) == select(k=0) == select(k=21) == select(G=-1) == _lib.ERR_SHAPE
    assert select(W=33, V=100) == select(k=65, V=100) == _lib.ERR_UNSUPPORTED
    assert select(G=40000) == _lib.ERR_SHAPE
    assert select(dtype=3) == _lib.ERR_DTYPE
    assert select(x=None) == select(ws=None) == select(ws_bytes=8) == select(stride=-1) == \
        select(x=p + 1) == select(ws=p + 8) == _lib.ERR_VALUE
    assert select(G=0) == 0
    def advance(G=1, W=2, k=4, T=3, E=1, alpha=1.0, first=p):
        return L.acorn_beam_advance(first, *[p] * 23, G, W, k, T, E, alpha, 0, 0, None)
    assert advance(W=0) == advance(k=0) == advance(T=0) == advance(E=-1) == _lib.ERR_SHAPE
    assert advance(W=33) == advance(k=65) == _lib.ERR_UNSUPPORTED
    assert advance(alpha=math.nan) == advance(first=None) == _lib.ERR_VALUE
    assert advance(G=0) == 0
    def reorder(G=1, W=2, ts=4, layers=1, NB=8, P=16, KV=2, D=64, esz=2, scales=None, k=p):
        return L.acorn_beam_reorder(k, p, scales, p, p, p, G, W, ts, layers, NB, P, KV, D, esz, None)
    assert reorder(ts=0) == reorder(layers=0) == reorder(P=0) == reorder(G=70000) == _lib.ERR_SHAPE
    assert reorder(W=33) == reorder(KV=1, D=4) == _lib.ERR_UNSUPPORTED
    assert reorder(esz=1) == _lib.ERR_DTYPE and reorder(scales=p) == _lib.ERR_SHAPE
    assert reorder(esz=1, scales=p, P=48) == reorder(esz=1, scales=p, P=8) == _lib.ERR_SHAPE
    assert reorder(esz=1, scales=p, D=32) == _lib.ERR_UNSUPPORTED
    assert reorder(k=None) == reorder(k=p + 8) == reorder(esz=1, scales=p + 8) == _lib.ERR_VALUE
    def trace(T=4, G=1, W=2, M=2, x=p):
        return L.acorn_beam_trace(x, p, p, p, p, T, G, W, M, 0, None)
    assert trace(W=0) == trace(T=-1) == trace(M=-1) == _lib.ERR_SHAPE
    assert trace(W=33) == _lib.ERR_UNSUPPORTED and trace(x=None) == _lib.ERR_VALUE
    assert trace(T=0) == trace(G=0) == trace(M=0) == 0


# ---- selection --------------------------------------------------------------------------------


def _logits(rows, V, dtype, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = 2.0 * torch.randn(rows, V + pad, generator=g) + torch.randn(rows, 1, generator=g)
    for _ in range(8):
        x[torch.arange(rows), torch.randint(0, V, (rows,), generator=g)] += 7.0
    scores = -12.0 * torch.rand(rows, generator=g)
    return x.to(dtype), scores


def _hold(x, scores, k, out=None):
    """beam_select on the GPU against the oracle."""
    got = out or _beam().beam_select(x.cuda() if not x.is_cuda else x, scores.cuda(), k)
    want = ref.select_ref(x, scores, k)
    assert torch.equal(got.status.cpu().long(), want[3])
    assert torch.equal(got.beam.cpu().long(), want[1])
    assert torch.equal(got.token.cpu(), want[2])
    s = got.score.cpu().double()
    fine = want[0] > -INF
    assert torch.equal(fine, s > -INF)
    assert ((s - want[0]).abs()[fine] <= score_bound(want[0], x.shape[1])[fine]).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G,W,V,k", [(1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 21), (3, 4, 1000, 8),
                                     (1, 32, 77, 64), (2, 5, 4097, 15), (5, 2, 8193, 1),
                                     (1, 4, 32768, 12), (70, 3, 517, 6), (130, 4, 20003, 8),
                                     (300, 4, 6001, 8)])
def test_select(dtype, G, W, V, k):
    x, s = _logits(G * W, V, dtype, G + V)
    _hold(x, s.view(G, W), k)


@gpu
@pytest.mark.parametrize("rows,W,k", [(1, 1, 2), (4, 4, 8), (64, 8, 64)])
def test_select_over_a_vocabulary(rows, W, k):
    x, s = _logits(rows, 151936, torch.bfloat16, rows)
    _hold(x, s.view(-1, W), k)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_select_of_rows_anywhere(dtype):
    """Rows inside a wider product, from any element on, the same row for every beam, columns apart."""
    V, k = 2051, 9
    x, s = _logits(6, V, dtype, 3, pad=13)
    wide, s = x.cuda(), s.view(2, 3)
    for first in (0, 1, 3, 13):
        _hold(wide[:, first:first + V], s, k)
    _hold(wide[:1, :V].expand(6, V), s, k)
    _hold(wide[:, :V].t().contiguous().t(), s, k)


@gpu
def test_equal_rows_tie_by_beam_then_token():
    """Beams of equal scores and equal logits, at addresses of every alignment: in turn by beam."""
    for V in (37, 4099, 20001):
        x, _ = _logits(1, V, torch.bfloat16, V)
        x = x.expand(4, V).contiguous()
        got = _beam().beam_select(x.cuda(), torch.full((1, 4), -3.0, device="cuda"), 16)
        order = torch.sort(x[0].double(), descending=True, stable=True)[1]
        flat = sorted(((-float(x[0, t]), b, int(t)) for b in range(4) for t in order[:16]))[:16]
        assert list(zip(got.beam[0].tolist(), got.token[0].tolist())) == [f[1:] for f in flat]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ["equal", "rising", "falling", "two", "zeros"])
def test_select_of_ordered_and_equal_logits(dtype, shape):
    V, k = 9001, 40
    i = torch.arange(V)
    row = {"equal": torch.full((V,), 1.5), "rising": i / 1000.0, "falling": -i / 1000.0,
           "two": (i % 2).float(), "zeros": torch.where(i % 3 == 0, -0.0, 0.0)}[shape].to(dtype)
    x = torch.stack([row, row, row])
    _hold(x, torch.tensor([[-1.0, -1.0, -2.5]]), k)


@gpu
@pytest.mark.parametrize("shape", ["equal", "rising"])
@pytest.mark.parametrize("G,W,V", [(300, 4, 6001), (130, 4, 20003)])
def test_select_of_ordered_and_equal_logits_in_many_rows(shape, G, W, V):
    """Long pieces, whose candidates do not fit where they are held."""
    i = torch.arange(V)
    row = (torch.full((V,), 1.5) if shape == "equal" else i / 100.0).to(torch.bfloat16)
    x = row.expand(G * W, V)
    s = -torch.arange(G * W).view(G, W) / 64.0
    _hold(x, s, 33)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_select_with_banned_tokens_and_dead_beams(dtype):
    """Fewer live continuations than k: those of -inf follow by beam and token. A row at the type's
    lowest value is an even distribution; one all banned has none; dead beams' rows are not read."""
    G, W, V, k = 4, 3, 300, 20
    x, s = _logits(G * W, V, dtype, 8)
    s = s.view(G, W)
    x[0, :] = -INF                       # group 0: a beam that may not go on
    x[1, 7:] = -INF                      # ... and one of 7 tokens
    x[2, 3:] = -INF
    low = torch.finfo(dtype).min
    x[3, :] = low                        # group 1: all at the lowest value
    x[4, 2:] = low
    s[1, 2] = -INF
    x[5] = math.nan                      # (not read)
    s[2, :] = -INF                       # group 2: nothing alive
    x[6:9] = INF
    big = torch.finfo(dtype).max
    x[9, 5], x[9, 6] = big, big          # group 3: the largest numbers
    _hold(x, s, k)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [math.nan, INF, -math.nan])
@pytest.mark.parametrize("where", [0, 4098])
def test_broken_rows_are_reported(dtype, value, where):
    x, s = _logits(6, 4099, dtype, 9)
    x[1, where] = value
    _hold(x, s.view(2, 3), 12)


@gpu
@pytest.mark.parametrize("value", [math.nan, INF])
def test_broken_scores_are_reported(value):
    x, s = _logits(6, 500, torch.bfloat16, 9)
    s[4] = value
    _hold(x, s.view(2, 3), 12)


@gpu
def test_select_into_buffers_on_a_stream_and_in_a_graph():
    b = _beam()
    x, s = _logits(8, 33001, torch.bfloat16, 10)
    x, s = x.cuda(), s.view(2, 4).cuda()
    out = b.beam_select(x, s, 8)
    ws = b.beam_select_workspace(2, 4, 33001, 8, x.dtype, "cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    mine = b.BeamCandidates(*(torch.empty_like(t) for t in out))
    with torch.cuda.stream(side):
        b.beam_select(x, s, 8, out=mine, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    _hold(x, s, 8, out=mine)
    assert graph_replays_match(lambda: b.beam_select(x, s, 8, out=mine, workspace=ws),
                               lambda: mine.token)
    assert graph_replays_match(lambda: b.beam_select(x, s, 8, out=mine, workspace=ws),
                               lambda: mine.score)
    with pytest.raises(AssertionError):
        b.beam_select(x, s, 8, out=mine, workspace=ws[:-8])
    with pytest.raises(ValueError):
        b.beam_select(x, s.cpu(), 8)
    none = b.beam_select(x[:0], s[:0], 8)
    assert none.token.shape == (0, 8)


# ---- bookkeeping ------------------------------------------------------------------------------


def _advance_case(G, W, K, T, E, seed, ending=0.3):
    g = torch.Generator().manual_seed(seed)

    def whole(lo, hi, *shape, dtype=torch.int32):
        return torch.randint(lo, hi, shape, generator=g).to(dtype)

    ends = torch.tensor([3, 7, 5][:E], dtype=torch.int64)
    token = whole(10, 40, G, K, dtype=torch.int64)
    if E:
        pick = ends[whole(0, E, G, K, dtype=torch.int64)]
        token = torch.where(torch.rand(G, K, generator=g) < ending, pick, token)
    score = (-5 - 10 * torch.rand(G, K, generator=g)).sort(-1, descending=True)[0]
    score[::3, K // 2:] = -INF                              # few candidates
    cand = {"score": score, "beam": whole(0, W, G, K), "token": token}
    held = torch.arange(W) < whole(0, W + 1, G, 1)
    old = (-1 - 2 * torch.rand(G, W, generator=g)).sort(-1, descending=True)[0]
    state = {"scores": -torch.rand(G, W, generator=g), "length": whole(0, T + 1, G),
             "done": whole(0, 5, G).eq(0).int(), "ids": whole(0, 9, G, W, dtype=torch.int64),
             "position": whole(0, 99, G, W), "parents": whole(0, W, G, W),
             "token_log": whole(0, 99, T, G, W), "parent_log": whole(0, W, T, G, W),
             "fin_scores": old.masked_fill(~held, -INF),
             "fin_length": whole(1, 9, G, W).masked_fill(~held, 0),
             "fin_beam": whole(0, W, G, W).masked_fill(~held, 0),
             "fin_token": whole(0, 9, G, W).masked_fill(~held, 0)}
    return state, cand, ends


@gpu
@pytest.mark.parametrize("early", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("G,W,K,E,alpha", [(1, 1, 1, 0, 1.0), (7, 1, 2, 1, 0.0), (9, 4, 8, 1, 1.0),
                                           (33, 5, 15, 2, 0.6), (6, 32, 64, 1, -1.0), (12, 8, 4, 3, 2.0)])
def test_advance(early, in_place, G, W, K, E, alpha):
    b = _beam()
    T = 6
    state, cand, ends = _advance_case(G, W, K, T, E, 100 * G + W)
    want = ref.advance_ref(state, cand, ends.tolist(), alpha, early, pad=99)
    st = b.BeamState(**{k: v.cuda() for k, v in state.items()})
    out = None if in_place else st._replace(**{k: torch.empty_like(v) for k, v in st._asdict().items()
                                               if not k.endswith("_log")})
    got = b.beam_advance(st, b.BeamCandidates(**{k: v.cuda() for k, v in cand.items()}), ends.cuda(),
                         length_penalty=alpha, early_stopping=early, pad=99, out=out)
    assert got is (st if in_place else out)
    for name, t in got._asdict().items():
        t = t.cpu()
        if name == "fin_scores":                            # one rounding to fp32
            fine = want[name] > -INF
            assert torch.equal(fine, t > -INF)
            assert ((t - want[name]).abs()[fine] <= 2.0 ** -24 * want[name].abs()[fine] * 1.001).all()
        else:
            assert torch.equal(t, want[name].to(t.dtype)), name


@gpu
def test_advance_in_a_graph():
    b = _beam()
    state, cand, ends = _advance_case(5, 4, 8, 6, 1, 1)
    st = b.BeamState(**{k: v.cuda() for k, v in state.items()})
    out = st._replace(**{k: torch.empty_like(v) for k, v in st._asdict().items()
                         if not k.endswith("_log")})
    cand = b.BeamCandidates(**{k: v.cuda() for k, v in cand.items()})
    ends = ends.cuda()
    for field in ("ids", "scores", "fin_scores"):
        assert graph_replays_match(lambda: b.beam_advance(st, cand, ends, out=out),
                                   lambda: getattr(out, field))


# ---- the cache follows ------------------------------------------------------------------------


def _reorder_case(G, W, P, lens, width, L, KV, D, dtype, seed):
    """A search's tables: shared full pages, then pages of each beam's own in every column."""
    g = torch.Generator().manual_seed(seed)
    NB = 6 + G * W * 3
    tables = torch.randint(0, 6, (G, 1, width), generator=g).repeat(1, W, 1).int()
    private = (torch.randperm(G * W * 3, generator=g) + 6).view(3, G, W).int()
    for n, tab, own in zip(lens, tables, private.permute(1, 0, 2)):
        for i in range(3):
            if n // P + i < width:
                tab[:, n // P + i] = own[i]
    if dtype == "8bit":
        pools = [torch.randint(0, 256, (L, NB, KV, P // 16, n), generator=g).to(torch.uint8)
                 for n in (16 * D, 16 * D, 32)]
    else:
        pools = [torch.randn(L, NB, P, KV, D, generator=g).to(dtype) for _ in range(2)]
    parents = torch.minimum(*torch.randint(0, W, (2, G, W), generator=g)).int()
    return pools, tables.reshape(G * W, width).contiguous(), \
        torch.tensor(lens, dtype=torch.int32)[:, None].repeat(1, W), parents


def _run_reorder(pools, tables, lens, parents):
    k, v, *scales = pools
    _beam().beam_reorder(k, v, tables, lens, parents, scale_pool=scales[0] if scales else None)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, "8bit"])
@pytest.mark.parametrize("W,P,lens", [(1, 16, (33, 48)), (2, 16, (0, 1, 15, 16, 17)), (4, 16, (300, 31)),
                                      (5, 32, (64, 65, 80, 81, 95)), (32, 64, (63, 1000)), (3, 16, (48,))])
def test_reorder(dtype, W, P, lens):
    """Groups at lengths from nothing to past the table's width, full pages among them."""
    width, L, KV, D = max(lens) // P + (0 if 48 in lens and W == 3 else 2), 3, 2, 64
    case = _reorder_case(len(lens), W, P, lens, width, L, KV, D, dtype, W)
    pools, tables, n, parents = case
    if W > 1:
        parents[0, 0], parents[-1, W - 1] = W, -1             # beams that there are not: themselves
    dev = [[p.cuda() for p in pools], tables.cuda(), n.cuda(), parents.cuda()]
    for _ in range(3):                                        # again on what it left
        ref.reorder_ref(pools, tables, n, parents, P, dtype == "8bit")
        _run_reorder(*dev)
        assert torch.equal(dev[1].cpu(), tables)
        for a, b in zip(dev[0], pools):
            assert torch.equal(a.cpu(), b)


@gpu
def test_reorder_of_pages_outside_the_pool_copies_nothing():
    pools, tables, n, parents = _reorder_case(1, 4, 16, (20,), 4, 2, 2, 64, torch.bfloat16, 3)
    parents[:] = 0
    tables[1, 1], tables[2, 1] = -5, pools[0].shape[1]
    dev = [[p.cuda() for p in pools], tables.cuda(), n.cuda(), parents.cuda()]
    ref.reorder_ref(pools, tables, n, parents, 16, False)
    _run_reorder(*dev)
    assert torch.equal(dev[1].cpu(), tables)
    for a, b in zip(dev[0], pools):
        assert torch.equal(a.cpu(), b)


@gpu
def test_reorder_in_a_graph():
    """Replays move the pages on from where the last one left them."""
    case = _reorder_case(3, 4, 16, (20, 40, 55), 5, 2, 2, 64, torch.bfloat16, 4)
    pools, tables, n, parents = case
    dev = [[p.cuda() for p in pools], tables.cuda(), n.cuda(), parents.cuda()]
    _run_reorder(*[[t.clone() for t in x] if isinstance(x, list) else x.clone() for x in dev])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _run_reorder(*dev)
    for step in range(4):
        gen = torch.Generator().manual_seed(step)
        parents = torch.randint(0, 4, (3, 4), generator=gen).int()
        dev[3].copy_(parents)
        g.replay()
        torch.cuda.synchronize()
        ref.reorder_ref(pools, tables, n, parents, 16, False)
        assert torch.equal(dev[1].cpu(), tables)
        for a, b in zip(dev[0], pools):
            assert torch.equal(a.cpu(), b)
        _ = torch.randn(1024, device="cuda").sum().item()


# ---- hypotheses -------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("T,G,W,M", [(1, 1, 1, 1), (2, 3, 4, 4), (15, 2, 3, 7), (16, 1, 32, 32),
                                     (17, 2, 5, 1), (250, 4, 8, 8), (1000, 1, 4, 70), (3001, 2, 2, 2)])
def test_trace(T, G, W, M):
    g = torch.Generator().manual_seed(T)
    tokens = torch.randint(0, 150000, (T, G, W), generator=g).int()
    parents = torch.minimum(*torch.randint(0, W, (2, T, G, W), generator=g)).int()
    steps = torch.randint(0, T + 1, (G, M), generator=g).int()
    steps[0, 0] = T
    if M > 3:
        steps[0, 1], steps[0, 2], steps[0, 3] = 0, -4, T + 9
    beams = torch.randint(0, W, (G, M), generator=g).int()
    if M > 4:
        beams[0, 4] = W
    got = _beam().beam_trace(tokens.cuda(), parents.cuda(), steps.cuda(), beams.cuda(), pad=-7)
    assert torch.equal(got.cpu(), ref.trace_ref(tokens, parents, steps, beams, pad=-7))


@gpu
def test_trace_of_logs_with_a_beam_that_there_is_not():
    tokens = torch.arange(40).view(20, 1, 2).int()
    parents = torch.zeros(20, 1, 2, dtype=torch.int32)
    parents[7, 0, 0] = 9
    steps, beams = torch.full((1, 1), 20).int(), torch.zeros(1, 1, dtype=torch.int32)
    got = _beam().beam_trace(tokens.cuda(), parents.cuda(), steps.cuda(), beams.cuda(), pad=-1)
    assert torch.equal(got.cpu(), ref.trace_ref(tokens, parents, steps, beams, pad=-1))
    assert got[0, 0, :7].tolist() == [-1] * 7 and got[0, 0, 7:].min() >= 0


@gpu
@pytest.mark.parametrize("least", [-2**31, -2**31 + 1, -1])
def test_trace_of_a_length_far_below_zero(least):
    tokens = torch.arange(80).view(40, 1, 2).int()
    parents = torch.zeros(40, 1, 2, dtype=torch.int32)
    steps, beams = torch.tensor([[least, 40]]).int(), torch.tensor([[1, 1]]).int()
    got = _beam().beam_trace(tokens.cuda(), parents.cuda(), steps.cuda(), beams.cuda(), pad=-1)
    assert torch.equal(got.cpu(), ref.trace_ref(tokens, parents, steps, beams, pad=-1))


def test_trace_refuses_logs_past_its_whole_numbers():
    from acorninfer_amd import _lib
    L, p = _lib.lib(), 64
    assert L.acorn_beam_trace(p, p, p, p, p, 2**30, 1, 1, 1, 0, None) == _lib.ERR_SHAPE
    assert L.acorn_beam_trace(p, p, p, p, p, 1, 2**27, 16, 1, 0, None) == _lib.ERR_SHAPE


def test_a_length_penalty_past_32_bits_is_refused():
    """Scores / steps ** penalty would be zeros, infinities or (0 / 0) NaN that have no order."""
    from acorninfer_amd import _lib
    from acorninfer_amd.ops import beam as b
    L, p = _lib.lib(), 64
    for steps, alpha, fits in ((4, 46.0, True), (4, 47.0, False), (4, -47.0, False), (2049, 8.3, True),
                               (2049, -8.4, False), (1, 1e300, True), (1, math.inf, False)):
        rc = L.acorn_beam_advance(*[p] * 24, 0, 2, 4, steps, 0, alpha, 0, 0, None)
        assert rc == 0                                      # (no groups: nothing to look at)
        if fits:
            b.check_length_penalty(alpha, steps)
            continue
        assert L.acorn_beam_advance(*[p] * 24, 1, 2, 4, steps, 0, alpha, 0, 0, None) == _lib.ERR_VALUE
        with pytest.raises(ValueError):
            b.check_length_penalty(alpha, steps)


@gpu
@pytest.mark.parametrize("T,G,W,M", [(600, 100, 4, 4), (600, 200, 4, 5), (2100, 130, 8, 8), (4500, 70, 32, 3),
                                     (1025, 65, 2, 2), (1030, 3, 4, 9)])
def test_trace_of_many_groups(T, G, W, M):
    """Batches whose groups are taken by one, two and four workgroups, stretches of 1 to 141 steps."""
    g = torch.Generator().manual_seed(T + G)
    tokens = torch.randint(0, 150000, (T, G, W), generator=g).int()
    parents = torch.randint(0, W, (T, G, W), generator=g).int()
    steps = torch.randint(T - 9, T + 1, (G, M), generator=g).int()
    steps[::7, 0] = torch.randint(0, T, (len(steps[::7]),), generator=g).int()
    beams = torch.randint(0, W, (G, M), generator=g).int()
    got = _beam().beam_trace(tokens.cuda(), parents.cuda(), steps.cuda(), beams.cuda(), pad=-7).cpu()
    want = torch.full((G, M, T), -7, dtype=torch.int64)       # (the oracle's steps, groups side by side)
    at, rows = beams.long(), torch.arange(G)[:, None]
    for t in range(T - 1, -1, -1):
        on = t < steps
        want[:, :, t] = torch.where(on, tokens[t][rows, at].long(), -7)
        at = torch.where(on, parents[t][rows, at].long(), at)
    assert torch.equal(got, want)
    assert torch.equal(want[:2], ref.trace_ref(tokens[:, :2], parents[:, :2], steps[:2], beams[:2], pad=-7))
