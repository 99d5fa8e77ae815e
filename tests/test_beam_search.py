"""A whole beam search (engine/beam.py): selection, bookkeeping, cache and hypotheses behind the
model's step, against oracle/beam_ref.search_ref over the CPU model and against the scores that
the model itself gives an answer read token by token."""
import math
from types import SimpleNamespace

import pytest
import torch

from acorninfer_amd.cache.pager import BlockAllocator, PagedCacheView, PagedKV8Cache, PagedKVCache
from acorninfer_amd.config import Qwen3Config
from oracle.beam_ref import search_ref

gpu = pytest.mark.gpu
TINY = Qwen3Config.tiny()
SMALL = Qwen3Config.qwen3_0_6b().with_layers(2)


def _search(model, num_blocks, eight=False, **kw):
    from acorninfer_amd.engine.beam import BeamSearch
    cfg = model.cfg
    alloc = BlockAllocator(num_blocks)
    cache = (PagedKV8Cache if eight else PagedKVCache)(
        cfg.num_hidden_layers, cfg.num_key_value_heads, cfg.head_dim, 16, alloc, model.device,
        model.dtype)
    return BeamSearch(model, cache, alloc, **kw), alloc


# ---- CPU ------------------------------------------------------------------------------------


def _host(**kw):
    """A BeamSearch without a model's weights: what it refuses, and its blocks."""
    from acorninfer_amd.engine.beam import BeamSearch
    model = SimpleNamespace(cfg=SMALL, device=torch.device("cpu"), kv8_page=lambda c: 0)
    alloc = BlockAllocator(kw.pop("blocks", 40))
    cache = SimpleNamespace(page_size=16, allocator=alloc)
    args = {"beams": 4, "max_tokens": 20, "max_model_len": 128, "eos_ids": {1}} | kw
    return BeamSearch(model, cache, alloc, **args), alloc


def test_refusals():
    for kw, err in (({"beams": 0}, ValueError), ({"max_tokens": 0}, ValueError),
                    ({"length_penalty": math.inf}, ValueError), ({"beams": 33}, NotImplementedError),
                    ({"beams": 22, "eos_ids": {1, 2}}, NotImplementedError)):
        with pytest.raises(err):
            _host(**kw)
    search, alloc = _host()
    for prompts, kw in (([], {}), ([[1], []], {}), ([[1]], {"max_tokens": 0}),
                        ([[1]], {"max_tokens": 21}), ([[1] * 120], {})):
        with pytest.raises(ValueError):
            search.search(prompts, **kw)
    alloc.assert_balanced()


@pytest.mark.parametrize("n,steps", [(1, 1), (15, 2), (16, 1), (16, 2), (17, 20), (31, 18), (48, 17)])
def test_blocks_of_a_search(n, steps):
    """Beams have pages of their own, all different, in every column that a token of the answer is
    written to (the last token is never written)."""
    search, alloc = _host()
    view = PagedCacheView(search.cache)
    own = []
    flat, room = search._reserve([n], [view], own, steps)
    rows, at = [], 0
    for r in room:
        rows.append(flat[at:at + r // 16])
        at += r // 16
    assert at == len(flat) and rows[0][:-(-n // 16)] == view.table
    for p in range(n, n + steps - 1):
        column = [r[p // 16] for r in rows]
        assert len(set(column)) == len(column) and min(column) >= 0
    if n % 16 and steps > 1:
        assert len({r[n // 16] for r in rows}) == 4
    assert sorted(own + view.table) == sorted({b for r in rows for b in r if b >= 0})


def test_a_search_that_does_not_fit_leaves_no_block():
    from acorninfer_amd.cache.pager import BlockExhausted
    search, alloc = _host(blocks=5)
    with pytest.raises(BlockExhausted):
        search.search([[1] * 40, [2] * 20])
    alloc.assert_balanced()


# ---- GPU ------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("capture", [False, True])
@pytest.mark.parametrize("beams,steps,alpha,early,ends", [
    (1, 9, 1.0, False, {1}), (4, 40, 1.0, False, {1, 9}), (5, 21, 0.0, True, set(range(0, 10))),
    (8, 18, 0.7, False, {1, 2, 3})])
def test_a_search_is_the_oracles(capture, beams, steps, alpha, early, ends):
    """fp32, three prompts of different lengths that end in, at and behind a page's border."""
    from acorninfer_amd.models.qwen3 import Qwen3DecodeModel, random_state_dict
    from oracle.qwen3_ref import Qwen3Ref
    sd = random_state_dict(TINY, seed=3, std=0.25, dtype=torch.float32)
    model = Qwen3DecodeModel.from_state_dict(TINY, sd, dtype=torch.float32, device="cuda")
    oracle = Qwen3Ref(TINY, sd, torch.float32)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 256, (n,), generator=g).tolist() for n in (5, 16, 31)]
    if beams * (len(ends) + 1) > 64:
        ends = set(list(ends)[:64 // beams - 1])
    search, alloc = _search(model, 300, beams=beams, max_tokens=steps, max_model_len=96,
                            eos_ids=ends, length_penalty=alpha, early_stopping=early, capture=capture)
    for _ in range(2):                                       # the second on what the first left
        got = search.search(prompts)
        alloc.assert_balanced()
        for prompt, hyps in zip(prompts, got):
            def logits_of(toks):
                return oracle.forward(torch.tensor([prompt + list(toks)]), oracle.new_cache())[0, -1]
            want = search_ref(logits_of, beams, steps, ends, alpha=alpha, early=early)
            assert [tuple(h.tokens) for h in hyps] == [w[1] for w in want]
            # (two fp32 models: logits of magnitude 10 differ by some 2^-19, sums over the steps)
            assert all(abs(h.score - w[0]) < 2.0 ** -12 for h, w in zip(hyps, want))
            assert all(h.ended == (h.tokens[-1] in ends) for h in hyps)


@gpu
@pytest.mark.parametrize("eight", [False, True])
def test_scores_are_what_the_model_gives_the_answer(eight):
    """bf16, both caches: an answer's score is the sum of the log-probabilities that decoding it token
    by token (through a cache of its own, another batch size) gives, within what bf16 logits of
    another rounding differ by; replays equal the launches one by one."""
    from acorninfer_amd.models.qwen3 import Qwen3DecodeModel, random_state_dict
    sd = random_state_dict(SMALL, seed=7, std=0.02, dtype=torch.bfloat16)
    model = Qwen3DecodeModel.from_state_dict(SMALL, sd, device="cuda")
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 151936, (n,), generator=g).tolist() for n in (20, 7)]
    answers = []
    for capture in (True, False):
        search, alloc = _search(model, 200, eight, beams=4, max_tokens=24, max_model_len=64,
                                eos_ids={151645}, capture=capture)
        answers.append(search.search(prompts))
        alloc.assert_balanced()
    assert answers[0] == answers[1]
    for prompt, hyps in zip(prompts, answers[0]):
        assert len(hyps) == 4 and [h.score for h in hyps] == sorted((h.score for h in hyps), reverse=True)
        for h in hyps[:2]:
            view = PagedCacheView(search.cache)
            logits = model.forward_prefill_batch(torch.tensor([prompt]).cuda(), [view],
                                                 real_lens=[len(prompt)])
            total, bound = 0.0, 0.0
            for tok in h.tokens:
                row = torch.log_softmax(logits[0].double(), -1)
                total += float(row[tok])
                # a bf16 logit is off by 2^-8 of its size at each side, and so is the sum of the others
                bound += 2.0 ** -6 * float(logits.abs().max()) + 2.0 ** -6
                logits = model.forward_decode(torch.tensor([[tok]]).cuda(), [view])
            assert abs(total - h.score * len(h.tokens)) <= bound
            for block in view.table:
                alloc.free(block)


@gpu
def test_an_engine_searches_between_its_steps():
    """Requests in flight go on as if there had been no search, and the blocks come back."""
    from acorninfer_amd.engine.engine import Engine
    from acorninfer_amd.models.qwen3 import Qwen3DecodeModel, random_state_dict
    from acorninfer_amd.sampler import SamplingParams
    sd = random_state_dict(SMALL, seed=7, std=0.02, dtype=torch.bfloat16)
    model = Qwen3DecodeModel.from_state_dict(SMALL, sd, device="cuda")
    prompt = list(range(100, 130))

    def run(search):
        eng = Engine(model, num_blocks=128, max_model_len=256)
        eng.submit(prompt, SamplingParams(temperature=0.0), max_tokens=12, eos_ids=frozenset())
        tokens, found = [], None
        for step in range(12):
            tokens += [o.token_id for o in eng.step()]
            if search and step == 5:
                found = eng.beam_search([prompt, prompt[:3]], beams=3, max_tokens=10, eos_ids=frozenset())
                again = eng.beam_search([prompt, prompt[:3]], beams=3, max_tokens=10, eos_ids=frozenset())
                assert found == again
        eng.assert_balanced()
        return tokens, found

    alone, _ = run(False)
    with_search, found = run(True)
    assert alone == with_search and len(alone) == 12
    assert [len(h) for h in found] == [3, 3] and all(len(h.tokens) == 10 for f in found for h in f)


@gpu
def test_a_prefill_after_a_search_reuses_its_buffers():
    """The model keeps the last prefill's buffers: a search's, which runs in inference mode, can be
    written outside it, and the other way round."""
    from acorninfer_amd.models.qwen3 import Qwen3DecodeModel, random_state_dict
    sd = random_state_dict(SMALL, seed=7, std=0.02, dtype=torch.bfloat16)
    model = Qwen3DecodeModel.from_state_dict(SMALL, sd, device="cuda")
    search, alloc = _search(model, 60, beams=2, max_tokens=3, max_model_len=64, eos_ids={1})
    prompt = list(range(50, 61))

    def prefill():
        view = PagedCacheView(search.cache)
        out = model.forward_prefill_batch(torch.tensor([prompt]).cuda(), [view], real_lens=[len(prompt)])
        for block in view.table:
            alloc.free(block)
        return out

    first = search.search([prompt])
    kept = model._extend_buf[1]
    logits = prefill()
    assert model._extend_buf[1] is kept
    assert search.search([prompt]) == first and model._extend_buf[1] is kept
    assert torch.equal(prefill(), logits)
    alloc.assert_balanced()


@gpu
def test_broken_logits_end_a_search():
    from acorninfer_amd.models.qwen3 import Qwen3DecodeModel, random_state_dict
    sd = random_state_dict(TINY, seed=3, std=0.25, dtype=torch.float32)
    sd["norm.weight"][5] = math.nan
    model = Qwen3DecodeModel.from_state_dict(TINY, sd, dtype=torch.float32, device="cuda")
    search, alloc = _search(model, 40, beams=2, max_tokens=4, max_model_len=64, eos_ids={1})
    with pytest.raises(ValueError):
        search.search([[3, 4, 5]])
    alloc.assert_balanced()


@gpu
def test_steps_of_many_sizes_and_settings_are_not_all_kept():
    """Searches over more numbers of prompts, and an engine's over more settings, than are kept: the
    first, made again, is what it was."""
    from acorninfer_amd.engine import beam, engine
    from acorninfer_amd.models.qwen3 import Qwen3DecodeModel, random_state_dict
    model = Qwen3DecodeModel.from_state_dict(TINY, random_state_dict(TINY, seed=3, std=0.25,
                                                                    dtype=torch.float32),
                                             dtype=torch.float32, device="cuda")
    search, alloc = _search(model, 200, beams=2, max_tokens=5, max_model_len=64, eos_ids={1})
    prompts = [[i + 3, 7, 20 - i] for i in range(beam.KEPT + 2)]
    first = search.search(prompts[:1])
    for n in range(2, len(prompts) + 1):
        assert len(search.search(prompts[:n])) == n
        assert len(search._batches) == min(n, beam.KEPT)
    assert search.search(prompts[:1]) == first
    assert list(search._batches) == [len(prompts) - 2, len(prompts) - 1, len(prompts), 1]
    alloc.assert_balanced()
    eng = engine.Engine(model, num_blocks=128, max_model_len=64)
    got = [eng.beam_search(prompts[:2], beams=2, max_tokens=5, length_penalty=i / 4, eos_ids=frozenset({1}))
           for i in (0, 1, 2, 3, 4, 5, 0)]
    assert got[0] == got[-1] and len(eng._searches) == engine.KEPT_SEARCHES
    eng.assert_balanced()


@gpu
@pytest.mark.parametrize("beams,prompts,steps", [(32, 3, 6), (4, 40, 5), (16, 70, 1)])
def test_searches_of_more_rows_than_an_engine_decodes(beams, prompts, steps):
    """96 to 1120 rows to a step, fp32 against the oracle, and all 32 beams."""
    from acorninfer_amd.models.qwen3 import Qwen3DecodeModel, random_state_dict
    from oracle.qwen3_ref import Qwen3Ref
    sd = random_state_dict(TINY, seed=3, std=0.25, dtype=torch.float32)
    model = Qwen3DecodeModel.from_state_dict(TINY, sd, dtype=torch.float32, device="cuda")
    oracle = Qwen3Ref(TINY, sd, torch.float32)
    g = torch.Generator().manual_seed(6)
    rows = [torch.randint(0, 256, (5 + i % 29,), generator=g).tolist() for i in range(prompts)]
    search, alloc = _search(model, 3000, beams=beams, max_tokens=6, max_model_len=64, eos_ids={1})
    got = search.search(rows, max_tokens=steps)
    alloc.assert_balanced()
    assert len(got) == prompts
    for i in (0, prompts // 2, prompts - 1):
        def logits_of(toks):
            return oracle.forward(torch.tensor([rows[i] + list(toks)]), oracle.new_cache())[0, -1]
        want = search_ref(logits_of, beams, steps, {1})
        assert [tuple(h.tokens) for h in got[i]] == [w[1] for w in want]
        assert all(abs(h.score - w[0]) < 2.0 ** -12 for h, w in zip(got[i], want))
