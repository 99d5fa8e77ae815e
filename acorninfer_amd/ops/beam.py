"""Beam search on the GPU: selection, bookkeeping, the cache and the answers.

A batch holds G groups (requests) of W beams; row g * W + w of a step's tensors is
beam w of group g. One step of a search, after the model's logits:

- `beam_select`   the k best continuations of every group
- `beam_advance`  the next beams and the finished hypotheses (a `BeamState`)
- `beam_reorder`  block tables and partly filled pages follow the beams
and at the end
- `beam_trace`    token rows out of the logs of tokens and parents

`engine.beam.BeamSearch` runs them behind the model's decode step, in one graph.
They stand beside the sampler (sampler.py) and the paged caches (cache/pager.py),
with the same block tables. Scores that are rounded to 32 bits at every step drift (by
0.1 in 2000 steps at sums of -15000): `low` operands carry what the rounding leaves out,
as BeamSearch does. Kernels: csrc/beam_select.hip, csrc/beam.hip. Up to 32
beams and 64 candidates. Everything launches on the current stream of its tensors'
device, never synchronises, and can be captured in a graph; calls that overlap must
not share outputs or a workspace.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple

import torch

from acorninfer_amd._lib import check, dtype_code, launch, lib, one_device, ptr

MAX_BEAMS = 32
MAX_CANDIDATES = 64
MAX_PENALTY = 64.0              # ln of the largest length ** length_penalty


class BeamCandidates(NamedTuple):
    """Continuations of every group, best first: score fp32, beam int32, token int64, [G, k]
    each; status int32 [G * W], 1 where a beam's score or logits hold NaN or +inf."""
    score: torch.Tensor
    beam: torch.Tensor
    token: torch.Tensor
    status: torch.Tensor | None = None


class BeamState(NamedTuple):
    """A search's state. [G, W]: scores (fp32, sums of log-probabilities; -inf: no such beam),
    ids (int64, the newest token), position (int32, the newest token's), parents (int32, the beam
    of the step before that it continues). [G] int32: length (tokens of the answer so far), done.
    [steps, G, W] int32: token_log, parent_log. The W best finished hypotheses, [G, W], best
    first: fin_scores (fp32, score / length ** penalty; -inf: none), fin_length (0: none),
    fin_token (the last token) and fin_beam (the beam of the step before that it continues)."""
    scores: torch.Tensor
    length: torch.Tensor
    done: torch.Tensor
    ids: torch.Tensor
    position: torch.Tensor
    parents: torch.Tensor
    token_log: torch.Tensor
    parent_log: torch.Tensor
    fin_scores: torch.Tensor
    fin_length: torch.Tensor
    fin_beam: torch.Tensor
    fin_token: torch.Tensor


_STATE_DTYPES = tuple({"scores": torch.float32, "fin_scores": torch.float32,
                       "ids": torch.int64}.get(n, torch.int32) for n in BeamState._fields)


def beam_state(groups: int, beams: int, steps: int, device, *,
               ids: torch.Tensor | None = None) -> BeamState:
    """A search that begins: beam 0 of every group at score 0, no others; room for `steps`
    tokens. `ids` [G, W] or [G * W] int64 contiguous: the buffer that a model's step reads."""
    assert groups >= 0 and beams >= 1 and steps >= 1
    if beams > MAX_BEAMS:
        raise NotImplementedError(f"{beams} beams: at most {MAX_BEAMS}")

    def z(*shape, dtype=torch.int32):
        return torch.zeros(*shape, dtype=dtype, device=device)

    state = BeamState(
        z(groups, beams, dtype=torch.float32), z(groups), z(groups),
        z(groups, beams, dtype=torch.int64) if ids is None else ids.view(groups, beams),
        z(groups, beams), z(groups, beams), z(steps, groups, beams), z(steps, groups, beams),
        z(groups, beams, dtype=torch.float32), *(z(groups, beams) for _ in range(3)))
    beam_reset(state)
    return state


def beam_reset(state: BeamState) -> None:
    """A state's buffers as `beam_state` makes them (the logs keep what they hold)."""
    for name, t in state._asdict().items():
        if not name.endswith("_log"):
            t.zero_()
    state.scores[:, 1:] = -math.inf
    state.fin_scores.fill_(-math.inf)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(groups: int, beams: int, vocab: int, k: int, dtype: int) -> int:
    n = ctypes.c_int64(0)
    check(lib().acorn_beam_select_workspace(groups, beams, vocab, k, dtype, ctypes.byref(n)),
          "beam_select_workspace")
    return n.value


def beam_select_workspace(groups: int, beams: int, vocab: int, k: int, dtype: torch.dtype,
                          device) -> torch.Tensor:
    """The workspace of a beam_select of these sizes."""
    code = dtype_code(torch.empty(0, dtype=dtype))
    return torch.empty(_workspace_bytes(groups, beams, vocab, k, code), dtype=torch.uint8,
                       device=device)


def _check(t: torch.Tensor, name: str, shape: tuple, dtype: torch.dtype) -> None:
    assert t.dtype is dtype and t.shape == shape and t.is_contiguous(), \
        f"{name} is contiguous {dtype} {list(shape)}, not {t.dtype} {list(t.shape)}"


def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: int, *,
                out: BeamCandidates | None = None, workspace: torch.Tensor | None = None,
                low: torch.Tensor | None = None, out_low: torch.Tensor | None = None
                ) -> BeamCandidates:
    """The k (at most 64) best continuations of every group by the beam's score plus the token's
    log-probability, compared in 64 bits; equal ones by beam and then token. (A row's sum of
    exponentials is good to 2e-7 as a rule: nearer scores of different beams come in the order of
    that error.) logits [G * W, V]
    fp32 / fp16 / bf16, rows any distance apart; scores [G, W] fp32. Tokens at -inf are banned; a
    beam of score -inf has only continuations of -inf, which come last (its logits are not read).
    A beam whose score or logits hold NaN or +inf counts as one of score -inf, and its status is
    1. `out` / `workspace` (beam_select_workspace of the same sizes) let a caller pass
    address-stable buffers. Scores in two words: `low` [G, W] fp32 is added to `scores`, `out_low`
    [G, k] fp32 gets what rounding the candidates' scores to fp32 left out."""
    assert scores.dim() == 2 and logits.dim() == 2, "scores are [G, W], logits [G * W, V]"
    G, W = scores.shape
    rows, V = logits.shape
    k = int(k)
    _check(scores, "scores", (G, W), torch.float32)
    assert rows == G * W and W >= 1 and V >= 1, f"{rows} rows of logits for {G} groups of {W} beams"
    assert 1 <= k <= W * V, f"k must be in 1 .. {W * V}, not {k}"
    if W > MAX_BEAMS or k > MAX_CANDIDATES:
        raise NotImplementedError(f"{W} beams, {k} candidates: at most {MAX_BEAMS} and "
                                  f"{MAX_CANDIDATES}")
    code = dtype_code(logits)
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    if out is None:
        dev = one_device(logits, scores)
        out = BeamCandidates(scores.new_empty((G, k)), scores.new_empty((G, k), dtype=torch.int32),
                             scores.new_empty((G, k), dtype=torch.int64),
                             scores.new_empty((G * W,), dtype=torch.int32))
    else:
        for name, dtype in (("score", torch.float32), ("beam", torch.int32), ("token", torch.int64)):
            _check(getattr(out, name), "out." + name, (G, k), dtype)
        assert out.status is not None
        _check(out.status, "out.status", (G * W,), torch.int32)
        dev = one_device(logits, scores, *out)
    need = _workspace_bytes(G, W, V, k, code)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=logits.device)
    else:
        assert workspace.get_device() == dev and workspace.is_contiguous() and \
            workspace.numel() * workspace.element_size() >= need and \
            workspace.data_ptr() % 16 == 0, "workspace: beam_select_workspace of the same sizes"
    if low is None and out_low is None:
        launch("beam_select", dev, logits.data_ptr(), logits.stride(0), scores.data_ptr(), G, W, V, k,
               out.score.data_ptr(), out.beam.data_ptr(), out.token.data_ptr(), out.status.data_ptr(),
               workspace.data_ptr(), workspace.numel() * workspace.element_size(), code)
        return out
    for name, t, n in (("low", low, W), ("out_low", out_low, k)):
        if t is not None:
            _check(t, name, (G, n), torch.float32)
            one_device(logits, t)
    launch("beam_select_low", dev, logits.data_ptr(), logits.stride(0), scores.data_ptr(), ptr(low),
           G, W, V, k, out.score.data_ptr(), ptr(out_low), out.beam.data_ptr(), out.token.data_ptr(),
           out.status.data_ptr(), workspace.data_ptr(), workspace.numel() * workspace.element_size(),
           code)
    return out


# (a state is twelve tensors, and a call looks at two of them: what is as it should be is passed in
# one expression, and only what is not is looked at field by field)
def _check_state(s: BeamState, name: str, G: int, W: int) -> None:
    scores, length, done, ids, position, parents, tlog, plog, fs, fl, fb, ft = s
    gw, g, log, i32, f32 = (G, W), (G,), (s.token_log.shape[0], G, W), torch.int32, torch.float32
    if scores.dtype is f32 is fs.dtype and ids.dtype is torch.int64 and length.dtype is i32 and \
            done.dtype is i32 and position.dtype is i32 and parents.dtype is i32 and \
            tlog.dtype is i32 and plog.dtype is i32 and fl.dtype is i32 and fb.dtype is i32 and \
            ft.dtype is i32 and scores.shape == gw == fs.shape == ids.shape == position.shape == \
            parents.shape == fl.shape == fb.shape == ft.shape and length.shape == g == done.shape and \
            tlog.shape == log == plog.shape and log[0] >= 1 and scores.is_contiguous() and \
            length.is_contiguous() and done.is_contiguous() and ids.is_contiguous() and \
            position.is_contiguous() and parents.is_contiguous() and tlog.is_contiguous() and \
            plog.is_contiguous() and fs.is_contiguous() and fl.is_contiguous() and \
            fb.is_contiguous() and ft.is_contiguous():
        return
    for field, t, dtype in zip(BeamState._fields, s, _STATE_DTYPES):
        shape = g if field in ("length", "done") else log if field.endswith("_log") else gw
        _check(t, f"{name}.{field}", shape, dtype)
    raise AssertionError("logs are [steps, G, W], of at least one step")


def check_length_penalty(alpha: float, steps: int) -> None:
    """Scores divided by steps ** alpha stay within 32 bits."""
    if not (math.isfinite(alpha) and abs(alpha) * math.log(steps) <= MAX_PENALTY):
        raise ValueError(f"length_penalty must be finite and at most {MAX_PENALTY} / ln({steps}) "
                         f"either way, not {alpha}")


def beam_advance(state: BeamState, candidates: BeamCandidates, end_ids: torch.Tensor, *,
                 length_penalty: float = 1.0, early_stopping: bool = False, pad: int = 0,
                 out: BeamState | None = None,
                 low: tuple[torch.Tensor, torch.Tensor] | None = None) -> BeamState:
    """One step of the bookkeeping: of a group's candidates (best first, at most 64) the first W
    that do not end (token in end_ids [E] int64) become its beams, row `length` of the logs holds
    their tokens and parents; those among the first W that end join the finished hypotheses, of
    which the W best by score / length ** length_penalty are kept. A group is done where no beam
    is left, where the logs are full, or where it has W finished hypotheses and (early_stopping,
    or its best beam's score / length ** length_penalty is no better than the worst of them).
    Groups that are done stay (ids `pad`, every beam its own parent). k = W * (E + 1) candidates
    are always enough for W beams; beams that get none have score -inf. |length_penalty| * ln(steps)
    is at most 64. Returns `out` (a state of the same sizes; by default `state`, in place), whose logs
    are written in place. Scores in two words, in place only: `low` = (the candidates' low words
    [G, K], the beams' [G, W], written), fp32."""
    assert state.scores.dim() == 2 and state.token_log.dim() == 3, \
        "scores are [G, W], logs [steps, G, W]"
    G, W = state.scores.shape
    out = state if out is None else out
    _check_state(state, "state", G, W)
    if out is not state:
        _check_state(out, "out", G, W)
        assert out.token_log.data_ptr() == state.token_log.data_ptr() and \
            out.parent_log.data_ptr() == state.parent_log.data_ptr() and \
            out.token_log.shape == state.token_log.shape, "the logs are one for all steps"
    score, beam, token = candidates[:3]
    assert score.dim() == 2 and score.shape[1] >= 1
    K, E = score.shape[1], end_ids.shape[0] if end_ids.dim() == 1 else -1
    _check(score, "candidates.score", (G, K), torch.float32)
    _check(beam, "candidates.beam", (G, K), torch.int32)
    _check(token, "candidates.token", (G, K), torch.int64)
    assert E >= 0 and end_ids.dtype is torch.int64 and end_ids.is_contiguous(), \
        "end_ids are contiguous int64 [E]"
    alpha = float(length_penalty)
    check_length_penalty(alpha, state.token_log.shape[0])
    if W > MAX_BEAMS or K > MAX_CANDIDATES:
        raise NotImplementedError(f"{W} beams, {K} candidates: at most {MAX_BEAMS} and "
                                  f"{MAX_CANDIDATES}")
    dev = one_device(*state, score, beam, token, end_ids, *(() if out is state else out))
    s, o = state, out
    words = ()
    if low is not None:
        assert out is state and len(low) == 2, "scores in two words are advanced in place"
        words = tuple(low)
        for name, t, n in zip(("low[0]", "low[1]"), words, (K, W)):
            _check(t, name, (G, n), torch.float32)
        one_device(score, *words)
    launch("beam_advance_low" if words else "beam_advance", dev, *map(torch.Tensor.data_ptr, (
        s.scores, s.length, s.done, s.position, s.fin_scores, s.fin_length, s.fin_beam, s.fin_token,
        o.scores, o.length, o.done, o.ids, o.position, o.parents, o.fin_scores, o.fin_length,
        o.fin_beam, o.fin_token, o.token_log, o.parent_log, score, beam, token, end_ids, *words)),
        G, W, K, s.token_log.shape[0], E, alpha, int(bool(early_stopping)), int(pad))
    return out


def beam_reorder(k_pool: torch.Tensor, v_pool: torch.Tensor, tables: torch.Tensor,
                 lens: torch.Tensor, parents: torch.Tensor, *,
                 scale_pool: torch.Tensor | None = None) -> None:
    """Block tables and the cache follow the beams: beam w of a group continues beam
    parents[g, w] [G, W] int32. tables [G * W, pages] int32, in place: with n = lens[g, 0] tokens
    ([G, W] int32, the same for a group's beams) the columns before n // P become the parent's
    (full pages are shared); where the last page is partly filled, each beam needs one of its own:
    the first child of a beam takes its page, every further child the page of a beam without
    children, into which the n % P tokens are copied in all layers. The group's entries of that
    column differ from one another, and so do those of the columns behind it, which stay.
    k_pool, v_pool [layers, num_blocks, P, KV, D] in 16 or 32 bits; with scale_pool those of
    PagedKV8Cache."""
    assert tables.dim() == 2 and tables.shape[1] >= 1 and tables.dtype is torch.int32 and \
        tables.is_contiguous(), "tables are contiguous int32 [G * W, pages]"
    assert parents.dim() == 2
    G, W = parents.shape
    _check(parents, "parents", (G, W), torch.int32)
    _check(lens, "lens", (G, W), torch.int32)
    assert tables.shape[0] == G * W, f"{tables.shape[0]} table rows for {G} groups of {W} beams"
    assert k_pool.dim() == 5 or scale_pool is not None, "pools are [layers, num_blocks, P, KV, D]"
    assert k_pool.dim() == 5 and v_pool.shape == k_pool.shape and v_pool.dtype is k_pool.dtype and \
        k_pool.is_contiguous() and v_pool.is_contiguous(), "k and v pools are alike and contiguous"
    if scale_pool is None:
        L, NB, P, KV, D = k_pool.shape
        assert k_pool.dtype.is_floating_point and k_pool.element_size() in (2, 4), \
            f"a pool of {k_pool.dtype}"
        dev = one_device(k_pool, v_pool, tables, lens, parents)
    else:
        L, NB, KV, groups, n = k_pool.shape
        P, D = groups * 16, n // 16
        assert k_pool.dtype is torch.uint8 and n % 16 == 0
        _check(scale_pool, "scale_pool", (L, NB, KV, groups, 32), torch.uint8)
        dev = one_device(k_pool, v_pool, tables, lens, parents, scale_pool)
    if W > MAX_BEAMS:
        raise NotImplementedError(f"{W} beams: at most {MAX_BEAMS}")
    launch("beam_reorder", dev, k_pool.data_ptr(), v_pool.data_ptr(),
           None if scale_pool is None else scale_pool.data_ptr(), tables.data_ptr(),
           lens.data_ptr(), parents.data_ptr(), G, W, tables.shape[1], L, NB, P, KV, D,
           k_pool.element_size())


def beam_trace(token_log: torch.Tensor, parent_log: torch.Tensor, steps: torch.Tensor,
               beams: torch.Tensor, *, pad: int = 0, out: torch.Tensor | None = None
               ) -> torch.Tensor:
    """Token rows [G, M, T] int64 out of the logs [T, G, W] int32: row (g, m) holds the
    steps[g, m] tokens that end with beam beams[g, m] of step steps[g, m] - 1 ([G, M] int32 both;
    steps of 0 and less give an empty row), and `pad` behind them."""
    assert token_log.dim() == 3 and steps.dim() == 2
    T, G, W = token_log.shape
    M = steps.shape[1]
    _check(token_log, "token_log", (T, G, W), torch.int32)
    _check(parent_log, "parent_log", (T, G, W), torch.int32)
    _check(steps, "steps", (G, M), torch.int32)
    _check(beams, "beams", (G, M), torch.int32)
    assert W >= 1
    if W > MAX_BEAMS:
        raise NotImplementedError(f"{W} beams: at most {MAX_BEAMS}")
    if out is None:
        dev = one_device(token_log, parent_log, steps, beams)
        out = torch.empty((G, M, T), dtype=torch.int64, device=token_log.device)
    else:
        _check(out, "out", (G, M, T), torch.int64)
        dev = one_device(token_log, parent_log, steps, beams, out)
    launch("beam_trace", dev, token_log.data_ptr(), parent_log.data_ptr(), steps.data_ptr(),
           beams.data_ptr(), out.data_ptr(), T, G, W, M, int(pad))
    return out
