"""Beam search over the paged cache, its loop on the GPU.

`BeamSearch` prefills the prompts of a batch and then replays one captured step per
token: slot map -> Qwen3DecodeModel.step -> beam_select -> beam_advance -> the cache
follows (ops/beam.py, ops/request_maps.py). The host looks only for groups that are
done, every CHECK_EVERY steps, and reads the hypotheses at the end. The reference has
no beam search.

Blocks: the prompt's full pages are shared by a group's beams; each beam has pages of its
own from the first partly filled one on, taken for the whole answer before the search
begins, so that no step needs the allocator. They are returned when the search ends.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from acorninfer_amd.cache.pager import BlockExhausted, PagedCacheView
from acorninfer_amd.models.qwen3 import Qwen3DecodeModel, StepBuffers
from acorninfer_amd.ops.beam import (MAX_BEAMS, MAX_CANDIDATES, BeamCandidates, BeamState,
                                     beam_advance, beam_reset, beam_select, beam_select_workspace,
                                     beam_state, beam_trace, check_length_penalty)
from acorninfer_amd.ops.request_maps import SlotMap, block_tables, slot_map

WARMUP_STEPS = 2
CHECK_EVERY = 16
KEPT = 4                        # numbers of groups whose buffers and step are kept


@dataclass(frozen=True)
class Hypothesis:
    """An answer: its tokens (the end token included, where it has one) and the sum of their
    log-probabilities / len(tokens) ** length_penalty."""
    tokens: list[int]
    score: float
    ended: bool


@dataclass
class _Batch:
    """Buffers and the captured step of one number of groups."""
    buf: StepBuffers
    state: BeamState
    cand: BeamCandidates
    ws: torch.Tensor
    slots: SlotMap
    ones: torch.Tensor
    broken: torch.Tensor
    # scores are sums of thousands of terms: what their 32 bits leave out, of candidates and beams
    low: tuple[torch.Tensor, torch.Tensor]
    graph: torch.cuda.CUDAGraph | None = None


class BeamSearch:
    def __init__(self, model: Qwen3DecodeModel, cache, allocator, *, beams: int, max_tokens: int,
                 max_model_len: int, eos_ids, length_penalty: float = 1.0,
                 early_stopping: bool = False, capture: bool = True):
        """Searches of up to max_tokens tokens over prompts with prompt + max_tokens <=
        max_model_len; hypotheses end with a token of eos_ids."""
        eos = sorted(set(int(i) for i in eos_ids))
        if beams < 1 or max_tokens < 1:
            raise ValueError("beams and max_tokens must be >= 1")
        check_length_penalty(float(length_penalty), max_tokens + 1)
        self.candidates = beams * (len(eos) + 1)     # enough for `beams` that do not end
        if beams > MAX_BEAMS or self.candidates > MAX_CANDIDATES:
            raise NotImplementedError(f"{beams} beams with {len(eos)} end tokens: at most "
                                      f"{MAX_BEAMS} beams, {MAX_CANDIDATES} candidates")
        if self.candidates > model.cfg.vocab_size:
            raise ValueError(f"{self.candidates} candidates of {model.cfg.vocab_size} tokens")
        self.model, self.cache, self.allocator = model, cache, allocator
        self.beams, self.max_tokens, self.max_model_len = beams, max_tokens, max_model_len
        self.penalty, self.early, self.capture = float(length_penalty), bool(early_stopping), capture
        self.device = model.device
        self.page = cache.page_size
        self.width = -(-max_model_len // self.page)
        self.end_ids = torch.tensor(eos, dtype=torch.int64, device=self.device)
        self._kv8 = model.kv8_page(cache)
        self._batches: dict[int, _Batch] = {}

    # ------------------------------------------------------------- one step --
    def _batch(self, G: int) -> _Batch:
        b = self._batches.pop(G, None)
        if b is None:
            while len(self._batches) >= KEPT:                # the one that was used longest ago
                torch.cuda.synchronize(self.device)          # (a search that was broken off may still run)
                del self._batches[next(iter(self._batches))]
            W, K, V, dev = self.beams, self.candidates, self.model.cfg.vocab_size, self.device
            B = G * W
            buf = self.model.buffers(B, self.width, kv8_page=self._kv8)
            # (one step more than a search takes: logs that are full would end a group)
            state = beam_state(G, W, self.max_tokens + 1, dev, ids=buf.ids)

            def z(*shape, dtype=torch.int32):
                return torch.zeros(*shape, dtype=dtype, device=dev)

            cand = BeamCandidates(z(G, K, dtype=torch.float32), z(G, K), z(G, K, dtype=torch.int64),
                                  z(B))
            b = _Batch(
                buf, state, cand, beam_select_workspace(G, W, V, K, buf.logits.dtype, dev),
                SlotMap(z(B), buf.positions, buf.pages, buf.slots, buf.lens, z(B)), z(B) + 1, z(B),
                (z(G, K, dtype=torch.float32), z(G, W, dtype=torch.float32)))
        self._batches[G] = b
        return b

    def _advance(self, b: _Batch, cand: BeamCandidates) -> None:
        beam_advance(b.state, cand, self.end_ids, length_penalty=self.penalty,
                     early_stopping=self.early, low=b.low)
        self.cache.reorder_beams(b.buf.tables, b.state.position, b.state.parents)

    def _body(self, b: _Batch) -> None:
        c = self.cache
        B = b.buf.batch
        slot_map(b.buf.tables, b.state.position.view(B), b.ones, self.page, B, out=b.slots)
        self.model.step(b.buf, c.k_pool, c.v_pool, c.num_blocks, self.page, sample=False,
                        scale_pool=c.scale_pool)
        beam_select(b.buf.logits, b.state.scores, self.candidates, out=b.cand, workspace=b.ws,
                    low=b.low[1], out_low=b.low[0])
        torch.maximum(b.broken, b.cand.status, out=b.broken)
        self._advance(b, b.cand)

    def _capture(self, b: _Batch) -> None:
        """Record the step; its warm-up runs on groups that are done, under tables without blocks, so
        that no cache row is written."""
        beam_reset(b.state)
        b.state.done.fill_(1)
        b.buf.tables.fill_(-1)
        s = torch.cuda.Stream(self.device)
        s.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(s):
            for _ in range(WARMUP_STEPS):
                self._body(b)
        torch.cuda.current_stream(self.device).wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self._body(b)
        b.graph = graph

    # ------------------------------------------------------------- a search --
    def _reserve(self, lens: list[int], views: list[PagedCacheView], own: list[int],
                 steps: int) -> tuple[list[int], list[int]]:
        """Block lists of every (group, beam), flat, and the tokens each has room for."""
        flat, room = [], []
        P = self.page
        for n, view in zip(lens, views):
            view._grow_to(-(-n // P))
            first, last = n // P, -(-(n + steps - 1) // P)   # columns that the beams write
            for w in range(self.beams):
                # (the columns before are beam 0's for all, from the first step on)
                row = list(view.table) if w == 0 else [-1] * first
                while len(row) < last:
                    row.append(self.allocator.allocate())
                    own.append(row[-1])
                flat += row
                room.append(len(row) * P)
        return flat, room

    @torch.inference_mode()
    def search(self, prompts: list[list[int]], *, max_tokens: int | None = None
               ) -> list[list[Hypothesis]]:
        """The best hypotheses of every prompt, at most `beams`, best first: those that ended, and
        where a search reached max_tokens with beams that may still win, these. BlockExhausted
        where the allocator cannot hold the search."""
        steps = self.max_tokens if max_tokens is None else int(max_tokens)
        if not prompts or any(not p for p in prompts):
            raise ValueError("prompts must be non-empty")
        if not 1 <= steps <= self.max_tokens:
            raise ValueError(f"max_tokens must be in 1 .. {self.max_tokens}")
        lens = [len(p) for p in prompts]
        if max(lens) + steps > self.max_model_len:
            raise ValueError(f"prompt + max_tokens ({max(lens) + steps}) exceeds max_model_len "
                             f"({self.max_model_len})")
        own: list[int] = []
        views = [PagedCacheView(self.cache) for _ in prompts]
        try:
            flat, room = self._reserve(lens, views, own, steps)
            with torch.cuda.device(self.device):
                return self._search(prompts, lens, views, flat, room, steps)
        finally:
            for block in own + [b for v in views for b in v.table]:
                self.allocator.free(block)

    def _search(self, prompts, lens, views, flat, room, steps) -> list[list[Hypothesis]]:
        G, W, dev = len(prompts), self.beams, self.device
        b = self._batch(G)
        if self.capture and b.graph is None:
            self._capture(b)
        beam_reset(b.state)
        b.broken.zero_()
        meta = torch.tensor(flat + room + [n - 1 for n in lens for _ in range(W)],
                            dtype=torch.int32).to(dev)
        n = len(flat)
        block_tables(meta[:n], meta[n:n + G * W], self.page, self.width, pad=-1,
                     out=b.buf.tables)
        b.state.position.copy_(meta[n + G * W:].view(G, W))

        # the prompts: one row of logits per group, whose best tokens are the first beams
        ids = torch.zeros(G, max(lens), dtype=torch.int64)
        for i, p in enumerate(prompts):
            ids[i, :len(p)] = torch.tensor(p, dtype=torch.int64)
        logits = self.model.forward_prefill_batch(ids.to(dev), views, real_lens=lens)
        zero = torch.zeros(G, 1, dtype=torch.float32, device=dev)
        cand = beam_select(logits, zero, self.candidates, out_low=b.low[0])
        b.broken[:G] = torch.maximum(b.broken[:G], cand.status)
        self._advance(b, cand)
        for t in range(1, steps):
            if t % CHECK_EVERY == 0 and bool((b.state.done != 0).all()):
                break
            if b.graph is not None:
                b.graph.replay()
            else:
                self._body(b)
        return self._hypotheses(b)

    def _hypotheses(self, b: _Batch) -> list[list[Hypothesis]]:
        s = b.state
        G, W = s.scores.shape
        # finished ones end behind their beam of the step before, the beams with their own
        at = torch.arange(W, dtype=torch.int32, device=self.device).expand(G, W)
        rows = beam_trace(s.token_log, s.parent_log,
                          torch.cat([s.fin_length - 1, s.length[:, None].expand(G, W)], 1).contiguous(),
                          torch.cat([s.fin_beam, at], 1).contiguous()).tolist()
        if int(b.broken.max()) != 0:
            raise ValueError("logits contain NaN/inf; model forward is broken")
        length, done = s.length.tolist(), s.done.tolist()
        scores = (s.scores.double() + b.low[1].double()).tolist()
        fin = [t.tolist() for t in (s.fin_scores, s.fin_length, s.fin_token)]
        answers = []
        for g in range(G):
            hyps = [Hypothesis(rows[g][m][:n - 1] + [last], score, True)
                    for m, (score, n, last) in enumerate(zip(*(f[g] for f in fin))) if n > 0]
            if not done[g]:
                hyps += [Hypothesis(rows[g][W + w][:length[g]], sc / length[g] ** self.penalty, False)
                         for w, sc in enumerate(scores[g]) if sc > -math.inf]
            answers.append(sorted(hyps, key=lambda h: -h.score)[:W])
        return answers


__all__ = ["BeamSearch", "BlockExhausted", "Hypothesis"]
