"""How exact the sums of a beam search are (ops/beam.py, engine/beam.py): scores of thousands of steps,
kept in two words, and a selection's sum of exponentials. Bounds count roundings; oracle:
oracle/beam_ref.py in 64 bits."""
import math
from types import SimpleNamespace

import pytest
import torch

from oracle import beam_ref as ref

gpu = pytest.mark.gpu
INF = math.inf
# log2 e as the kernels' 32 bits hold it is 1.34e-8 too small; of a row's ln sum that leaves at most
# as much of its entropy
LOG2E_OFF = 1.34e-8


def _beam():
    from acorninfer_amd.ops import beam
    return beam


def _ln_sum_bound(vocab):
    """Of a row in pieces of two vectors a lane, whatever the vocabulary: pieces are added in 64 bits.
    In 2^-24 of the sum: a power 14 (1 ulp is 2, and its exponent's rounding 2^-24 |t| ln 2 e^t-weighted,
    |t| < 16), a vector's sum 7, a new maximum 5, the lane's sum 3, its last factor 3, lanes 6 + 6,
    waves 3 * 6; and the entropy's share."""
    return 2.0 ** -24 * 62 + LOG2E_OFF * math.log(vocab)


# ---- a selection's sum ------------------------------------------------------------------------


def _select(x, k, W=1):
    """(s in 64 bits, beam, token) of beams at score 0."""
    zero = torch.zeros(x.shape[0] // W, W, device="cuda")
    low = torch.empty(x.shape[0] // W, k, device="cuda")
    got = _beam().beam_select(x.cuda(), zero, k, out_low=low)
    assert int(got.status.max()) == 0
    return (got.score.double() + low.double()).cpu(), got.beam.cpu().long(), got.token.cpu()


@gpu
@pytest.mark.parametrize("dtype,tail", [(torch.bfloat16, -18.75), (torch.float16, -18.75),
                                        (torch.float32, -18.0625)])
def test_what_additions_round_off_is_kept(dtype, tail):
    """Rows with nearly all of their probability in one token, each of whose others that a lane meets,
    a vector of them at a time, is less than half a unit in the last place beside it. More than 1024
    rows, so that a lane's piece is the longest, 19 vectors; the lane differs from row to row."""
    E = 16 // dtype.itemsize
    rows, V = 1030, 19 * 256 * E
    lane = torch.arange(V) // E % 256
    x = torch.where(lane == torch.arange(rows)[:, None] % 256, tail, -INF)
    first = torch.arange(rows) % 256 * E + torch.arange(rows) % E
    x[torch.arange(rows), first] = 0.0
    s, _, token = _select(x.to(dtype), 1)
    assert torch.equal(token[:, 0], first)
    w = math.exp(tail)
    # what the peak's own vector drops, and the last rounding
    bound = (E - 1) * w + 2.0 ** -24
    assert E * w < 2.0 ** -24 and 18 * E * w > 5 * bound    # (lost without the compensation)
    assert ((s[:, 0] + math.log1p((19 * E - 1) * w)).abs() <= bound).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("value", [0.0, 1.5, -7.25])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 37), (2, 4099), (1, 151936), (300, 20003)])
def test_the_sum_of_even_rows(dtype, value, rows, V):
    """Every token's log-probability is -ln V: exactly, but for the entropy's share and ln's 1e-12, where
    the powers are 1. Else in 2^-24: a power 2, a vector's sum 7, the lane's 3, its last factor 3, lanes
    6, waves 3."""
    k = min(V, 5)
    s, _, token = _select(torch.full((rows, V), value, dtype=dtype), k)
    assert torch.equal(token, torch.arange(k).expand(rows, k))
    bound = LOG2E_OFF * math.log(V) + 1e-11 + (0.0 if value == 0 else 2.0 ** -24 * 24)
    assert ((s + math.log(V)).abs() <= bound).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,W,k", [(1, 1, 2), (4, 4, 8), (4, 1, 64), (8, 8, 33)])
@pytest.mark.parametrize("late", [False, True])
def test_rows_of_many_pieces(dtype, rows, W, k, late):
    """A vocabulary of 151936 in few rows: 38 pieces in 16 bits, 75 in 32, more than a wave of the
    join has lanes. late: a row's maximum and its best tokens are in the last ones."""
    V = 151936
    g = torch.Generator().manual_seed(rows + k)
    x = 2.0 * torch.randn(rows, V, generator=g) + torch.randn(rows, 1, generator=g)
    for _ in range(2 * k):
        at = torch.randint(140000 if late else 0, V, (rows,), generator=g)
        x[torch.arange(rows), at] = 8.0 + 6.0 * torch.rand(rows, generator=g)
    x = x.to(dtype)
    s, beam, token = _select(x, k, W)
    want = ref.select_ref(x, torch.zeros(rows // W, W), k)
    assert torch.equal(beam, want[1]) and torch.equal(token, want[2])
    assert not late or int(token[:, 0].min()) >= 140000
    assert ((s - want[0]).abs() <= _ln_sum_bound(V) + 2.0 ** -48 * want[0].abs()).all()


# ---- scores in two words ----------------------------------------------------------------------


def test_refusals_of_low_words():
    from acorninfer_amd import _lib
    b = _beam()
    x, s = torch.zeros(6, 10), torch.zeros(2, 3)
    for bad in ({"low": s.double()}, {"low": s[:1]}, {"low": torch.zeros(2, 4)}, {"out_low": s},
                {"out_low": torch.zeros(4, 2).t()}, {"low": s, "out_low": torch.zeros(2, 5)}):
        with pytest.raises((AssertionError, ValueError)):
            b.beam_select(x, s, 4, **bad)
    st = b.beam_state(2, 3, 4, "cpu")
    c = torch.zeros(2, 6)
    cand = b.BeamCandidates(c, c.int(), c.long())
    other = st._replace(scores=st.scores.clone())
    for bad in ({"low": (s, s)}, {"low": (c,)}, {"low": (c, s.double())}, {"low": (c, c)},
                {"low": (c, s), "out": other}):
        with pytest.raises((AssertionError, ValueError)):
            b.beam_advance(st, cand, torch.tensor([1]), **bad)
    L, p = _lib.lib(), 64                                   # a pointer that is never followed
    def select(W=2, dtype=2, x=p):
        return L.acorn_beam_select_low(x, 10, p, p, 1, W, 10, 4, p, p, p, p, p, p, 1 << 20, dtype, None)
    assert select(W=0) == _lib.ERR_SHAPE and select(dtype=3) == _lib.ERR_DTYPE
    assert select(x=None) == _lib.ERR_VALUE
    def advance(W=2, first=p):
        return L.acorn_beam_advance_low(first, *[p] * 25, 1, W, 4, 3, 1, 1.0, 0, 0, None)
    assert advance(W=0) == _lib.ERR_SHAPE and advance(first=None) == _lib.ERR_VALUE


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V,k", [(5, 8), (4097, 12)])
def test_select_of_scores_in_two_words(dtype, V, k):
    """Scores near -4000, where 32 bits are 2.4e-4 apart; of group 1 the same row for all beams, whose
    scores differ in their low words alone; of group 2 beams that are dead or broken."""
    b = _beam()
    G, W = 3, 4
    g = torch.Generator().manual_seed(V)
    x = (2.0 * torch.randn(G * W, V, generator=g)).to(dtype)
    scores = -4000.0 - 3.0 * torch.rand(G, W, generator=g)
    low = 1e-4 * (torch.rand(G, W, generator=g) - 0.5)
    x[W:2 * W], scores[1] = x[W].clone(), -4000.0
    low[1] = torch.tensor([1e-5, 4e-5, -2e-5, 2e-5])
    scores[2, 0], low[2, 0], low[2, 2] = -INF, 0.0, math.nan
    out_low = torch.full((G, k), 7.0, device="cuda")
    got = b.beam_select(x.cuda(), scores.cuda(), k, low=low.cuda(), out_low=out_low)
    want = ref.select_ref(x, scores.double() + low.double(), k)
    assert torch.equal(got.status.cpu().long(), want[3]) and int(want[3].sum()) == 1
    assert torch.equal(got.beam.cpu().long(), want[1]) and torch.equal(got.token.cpu(), want[2])
    if V == 5:
        assert got.beam[1].tolist()[:4] == [1, 3, 0, 2]
    fine = want[0] > -INF
    hi, rest = got.score.cpu().double(), out_low.cpu().double()
    assert torch.equal(hi > -INF, fine) and (rest[~fine] == 0).all()
    bound = _ln_sum_bound(V) + 2.0 ** -48 * want[0].abs()    # (two words hold s to 2^-49)
    assert ((hi + rest - want[0]).abs() <= bound)[fine].all()
    assert (rest.abs() <= 2.0 ** -24 * hi.abs())[fine].all()
    assert torch.equal(hi.float(), (hi + rest).float())
    one = b.beam_select(x.cuda(), scores.cuda(), k, low=low.cuda())          # either alone
    assert torch.equal(one.score, got.score) and torch.equal(one.token, got.token)
    none = torch.full_like(out_low, 7.0)
    plain = b.beam_select(x.cuda(), scores.cuda(), k, out_low=none)
    zero = b.beam_select(x.cuda(), scores.cuda(), k, low=torch.zeros_like(low).cuda())
    assert torch.equal(plain.score, zero.score) and torch.equal(plain.token, zero.token)
    assert torch.equal(plain.score, b.beam_select(x.cuda(), scores.cuda(), k).score)
    assert (none[plain.score > -INF] != 7.0).all()


@gpu
@pytest.mark.parametrize("G,W,K,alpha", [(9, 4, 8, 1.0), (6, 32, 64, 0.0), (7, 1, 2, 0.6)])
def test_advance_of_scores_in_two_words(G, W, K, alpha):
    """The low words follow their candidates, finished hypotheses are divided from both words, groups
    that are done keep theirs."""
    b = _beam()
    g = torch.Generator().manual_seed(W)
    T, ends = 3000, torch.tensor([3])
    token = torch.randint(3, 6, (G, K), generator=g)
    exact = (-9000.0 - 20.0 * torch.rand(G, K, generator=g, dtype=torch.float64)).sort(-1, descending=True)[0]
    exact[2, K // 2:] = -INF
    score = exact.float()
    low = torch.where(exact > -INF, exact - score.double(), 0.0).float()
    cand = {"score": score.double() + low.double(), "token": token,
            "beam": torch.randint(0, W, (G, K), generator=g, dtype=torch.int32)}
    state = b.beam_state(G, W, T, "cpu")
    state.length.fill_(2500)
    state.done[1] = 1
    want = ref.advance_ref(state._asdict(), cand, [3], alpha, False)
    dev = b.BeamState(*(t.cuda() for t in state))
    words = (low.cuda(), torch.full((G, W), 5.0, device="cuda"))
    b.beam_advance(dev, b.BeamCandidates(score.cuda(), cand["beam"].cuda(), token.cuda()), ends.cuda(),
                   length_penalty=alpha, low=words)
    for name in ("ids", "parents", "length", "done", "fin_length", "fin_beam", "fin_token"):
        assert torch.equal(getattr(dev, name).cpu(), want[name].to(getattr(dev, name).dtype)), name
    assert torch.equal(dev.scores.cpu(), want["scores"])
    fine = want["fin_scores"] > -INF
    off = (dev.fin_scores.cpu() - want["fin_scores"]).abs()
    assert (off <= 2.0 ** -24 * 1.001 * want["fin_scores"].abs())[fine].all()
    for i in range(G):
        if i == 1:
            assert (words[1][i] == 5.0).all()
            continue
        goes = [float(l) for s, l, t in zip(score[i], low[i], token[i]) if s > -INF and t != 3][:W]
        assert words[1][i].tolist() == goes + [0.0] * (W - len(goes))


# ---- long searches ----------------------------------------------------------------------------

ROWS, VOCAB = 64, 4096


class Bigram:
    """What a search asks of a model, with logits that depend on the newest token alone."""

    def __init__(self, table):
        self.table, self.device, self.dtype = table.cuda(), torch.device("cuda", 0), table.dtype
        self.cfg = SimpleNamespace(vocab_size=table.shape[1])

    def kv8_page(self, cache):
        return 0

    def buffers(self, batch, width, kv8_page=0):
        def z(*shape, dtype=torch.int64):
            return torch.zeros(*shape, dtype=dtype, device="cuda")
        return SimpleNamespace(batch=batch, ids=z(batch), positions=z(batch), pages=z(batch),
                               slots=z(batch), lens=z(batch, dtype=torch.int32),
                               tables=z(batch, width, dtype=torch.int32),
                               logits=z(batch, self.table.shape[1], dtype=self.dtype))

    def step(self, buf, k_pool, v_pool, num_blocks, page, *, sample, scale_pool):
        buf.logits.copy_(self.table[buf.ids % ROWS])

    def forward_prefill_batch(self, ids, views, *, real_lens):
        last = ids[torch.arange(len(views)), torch.tensor(real_lens) - 1]
        return self.table[last % ROWS].float()


def _table(even):
    """even: all tokens that are not banned alike, so that powers are 1 and their sum exact. Else
    twelve tokens of a row above the rest."""
    g = torch.Generator().manual_seed(11)
    t = torch.zeros(ROWS, VOCAB)
    if even:
        share = 0.3 + 0.7 * torch.rand(ROWS, 1, generator=g)
        return t.masked_fill(torch.rand(ROWS, VOCAB, generator=g) >= share, -INF)
    at = torch.rand(ROWS, VOCAB, generator=g).argsort(-1)[:, :12]
    return t.scatter(1, at, 0.5 + 1.5 * torch.rand(ROWS, 12, generator=g))


def _step_bound(even):
    """What a step adds to a score's error. Even rows: the entropy's share; all else is below 1e-11 (ln
    to 1e-12, scores of 2^14 in 48 bits). Others, in 2^-24 of the sum: a power 4 (1 ulp, and its exponent
    below 4), a vector's sum 3, a new maximum 5, the lane's sum 3, its last factor 3, lanes 6 + 6, waves
    3 * 7, and the even row's."""
    return LOG2E_OFF * math.log(VOCAB) + (1e-11 if even else 2.0 ** -24 * 51)


@gpu
@pytest.mark.parametrize("capture", [False, True])
@pytest.mark.parametrize("even,beams", [(True, 1), (False, 3)])
def test_scores_of_long_searches(even, beams, capture):
    """2000 steps, scores to -15700: a sum held in 32 bits between steps would be 0.09 to 0.14 off (each
    step rounds to 2^-11, and the paths' cycles repeat their roundings); the steps' own errors add
    up to 2.2e-4 and 6e-3. Where a beam is chosen scores are 9e-4 apart or more, and beams have all
    but a few steps in common."""
    from acorninfer_amd.cache.pager import BlockAllocator, PagedKVCache
    from acorninfer_amd.engine.beam import BeamSearch
    table, steps = _table(even), 2000
    alloc = BlockAllocator(1200)
    search = BeamSearch(Bigram(table), PagedKVCache(1, 1, 16, 16, alloc, torch.device("cuda", 0),
                                                    torch.float32), alloc, beams=beams,
                        max_tokens=steps, max_model_len=2048, eos_ids=(), length_penalty=0.0,
                        capture=capture)
    prompts = [[3, 5], [20], [8, 8, 37]]
    for prompt, got in zip(prompts, search.search(prompts)):
        want = ref.search_ref(lambda toks: table[(toks or prompt)[-1] % ROWS], beams, steps, (), alpha=0.0)
        assert [tuple(h.tokens) for h in got] == [w[1] for w in want]
        assert all(abs(h.score - w[0]) <= steps * _step_bound(even) for h, w in zip(got, want))
    alloc.assert_balanced()
