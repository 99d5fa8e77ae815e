"""Plain statements of beam search over a paged cache, on the CPU: selection in 64 bits,
bookkeeping, block tables and pages, hypotheses, request maps, and a whole search over a
function that gives logits. No counterpart in the reference."""
from __future__ import annotations

import math

import torch

INF = float("inf")


def select_ref(logits: torch.Tensor, scores: torch.Tensor, k: int):
    """(score fp64 [G, k], beam [G, k], token [G, k], status [G * W]) of logits [G * W, V] and
    scores [G, W]: falling, equal ones by beam and token."""
    G, W = scores.shape
    V = logits.shape[1]
    x = logits.double().cpu().view(G, W, V)
    s = scores.double().cpu()
    score, beam, token, status = [], [], [], []
    for g in range(G):
        y = torch.full((W, V), -INF, dtype=torch.float64)
        for w in range(W):
            row, sc = x[g, w], float(s[g, w])
            bad = math.isnan(sc) or sc == INF
            if sc > -INF and not bad:
                bad = bool(torch.isnan(row).any() or (row == INF).any())
                m = float(row.max())
                if not bad and m > -INF:
                    y[w] = sc + ((row - m) - math.log(float(torch.exp(row - m).sum())))
            status.append(int(bad))
        order = torch.sort(y.view(-1), descending=True, stable=True)[1][:k]
        score.append(y.view(-1)[order])
        beam.append(order // V)
        token.append(order % V)
    return torch.stack(score), torch.stack(beam), torch.stack(token), torch.tensor(status)


def advance_ref(state: dict, cand: dict, ends, alpha: float, early: bool, pad: int = 0) -> dict:
    """The state after one step, from tensors on the CPU (a copy; fin_scores in fp64)."""
    st = {k: v.clone() for k, v in state.items()}
    st["fin_scores"] = st["fin_scores"].double()
    G, W = st["scores"].shape
    T, K = st["token_log"].shape[0], cand["score"].shape[1]
    for g in range(G):
        t = int(st["length"][g])
        st["parents"][g] = torch.arange(W)
        st["ids"][g] = pad
        if int(st["done"][g]) or t >= T:
            continue
        held = [tuple(float(st[k][g, i]) if k == "fin_scores" else int(st[k][g, i])
                      for k in ("fin_scores", "fin_length", "fin_beam", "fin_token"))
                for i in range(W) if int(st["fin_length"][g, i]) > 0]
        st["scores"][g] = -INF
        n = 0
        for i in range(K):
            v, b, tok = float(cand["score"][g, i]), int(cand["beam"][g, i]), int(cand["token"][g, i])
            if not v > -INF or not 0 <= b < W:
                continue
            if tok in ends:
                if i < W:
                    held.append((v / (t + 1) ** alpha, t + 1, b, tok))
            elif n < W:
                st["scores"][g, n], st["parents"][g, n], st["ids"][g, n] = v, b, tok
                n += 1
        held.sort(key=lambda e: -e[0])
        held = held[:W]
        best = float(st["scores"][g, 0]) / (t + 1) ** alpha
        full = len(held) == W
        st["done"][g] = int(n == 0 or t + 1 >= T or (full and (early or held[-1][0] >= best)))
        held += [(-INF, 0, 0, 0)] * (W - len(held))
        for j, k in enumerate(("fin_scores", "fin_length", "fin_beam", "fin_token")):
            st[k][g] = torch.tensor([e[j] for e in held], dtype=st[k].dtype)
        st["length"][g] = t + 1
        st["position"][g] += 1
        st["token_log"][t, g] = st["ids"][g].int()
        st["parent_log"][t, g] = st["parents"][g].int()
    return st


def deal_pages(parents: list[int], page: list[int]) -> tuple[list[int], list[tuple[int, int]]]:
    """(the page of every next beam, copies as (from, to)) where the last page is partly filled."""
    W = len(parents)
    spare = [page[w] for w in range(W) if w not in parents]
    taken, copies, seen = [], [], set()
    for p in parents:
        if p not in seen:
            seen.add(p)
            taken.append(page[p])
        else:
            to = spare.pop(0)
            taken.append(to)
            copies.append((page[p], to))
    return taken, copies


def reorder_ref(pools: list[torch.Tensor], tables: torch.Tensor, lens: torch.Tensor,
                parents: torch.Tensor, page_size: int, tiles: bool) -> None:
    """In place, on the CPU. pools: [L, NB, P, KV, D], or with `tiles` [L, NB, KV, P // 16, n]."""
    G, W = parents.shape
    tab = tables.view(G, W, -1)
    for g in range(G):
        n = int(lens[g, 0])
        par = [p if 0 <= p < W else w for w, p in enumerate(parents[g].tolist())]
        c, fill = n // page_size, n % page_size
        old = tab[g].clone()
        tab[g, :, :c] = old[par, :c]
        if n <= 0 or fill == 0 or c >= tab.shape[2]:
            continue
        taken, copies = deal_pages(par, old[:, c].tolist())
        tab[g, :, c] = torch.tensor(taken, dtype=tab.dtype)
        for pool in pools:
            for src, dst in copies:
                if not (0 <= src < pool.shape[1] and 0 <= dst < pool.shape[1]):
                    continue
                if tiles:
                    m = -(-fill // 16)
                    pool[:, dst, :, :m] = pool[:, src, :, :m]
                else:
                    pool[:, dst, :fill] = pool[:, src, :fill]


def trace_ref(token_log, parent_log, steps, beams, pad: int = 0) -> torch.Tensor:
    T, G, W = token_log.shape
    M = steps.shape[1]
    out = torch.full((G, M, T), pad, dtype=torch.int64)
    for g in range(G):
        for m in range(M):
            b = int(beams[g, m])
            for t in range(min(int(steps[g, m]), T) - 1, -1, -1):
                if not 0 <= b < W:
                    break
                out[g, m, t] = int(token_log[t, g, b])
                b = int(parent_log[t, g, b])
    return out


def block_tables_ref(blocks, lengths, page_size: int, width: int, pad: int = 0) -> torch.Tensor:
    out = torch.full((len(lengths), width), pad, dtype=torch.int32)
    at = 0
    for n, length in enumerate(lengths.tolist()):
        own = -(-length // page_size) if length > 0 else 0
        row = blocks[at:at + own][:width]
        out[n, :len(row)] = row
        at += own
    return out


def slot_map_ref(tables, starts, counts, page_size: int, rows: int, into: list) -> list:
    """[seq, positions, pages, slots, lens, row0]: the first five filled into `into`."""
    r, row0 = 0, []
    for n, (s, c) in enumerate(zip(starts.tolist(), counts.tolist())):
        row0.append(r)
        for j in range(max(c, 0)):
            if r < rows:
                p = s + j
                page = int(tables[n, p // page_size]) if 0 <= p < tables.shape[1] * page_size else -1
                for x, v in zip(into, (n, p, page, p % page_size, p + 1)):
                    x[r] = v
            r += 1
    return into + [torch.tensor(row0, dtype=torch.int32)]


def search_ref(logits_of, beams: int, steps: int, ends, *, alpha: float = 1.0, early: bool = False):
    """A whole search: logits_of(tokens) -> [V] logits after the answer's tokens so far. Returns
    hypotheses (score / length ** alpha, tokens), best first, at most `beams`."""
    live, held = [(0.0, ())], []
    for t in range(steps):
        cand = []
        for b, (s, toks) in enumerate(live):
            row = torch.log_softmax(logits_of(toks).double(), -1)
            top = torch.sort(row, descending=True, stable=True)
            for v, i in zip(top[0][:beams * (len(ends) + 1)], top[1][:beams * (len(ends) + 1)]):
                cand.append((s + float(v), b, int(i)))
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        cand = cand[:beams * (len(ends) + 1)]
        nxt = []
        for i, (s, b, tok) in enumerate(cand):
            if not s > -INF:
                continue
            if tok in ends:
                if i < beams:
                    held.append((s / (t + 1) ** alpha, live[b][1] + (tok,)))
            elif len(nxt) < beams:
                nxt.append((s, live[b][1] + (tok,)))
        held = sorted(held, key=lambda h: -h[0])[:beams]
        live = nxt
        if not live or (len(held) == beams and (early or held[-1][0] >= live[0][0] / (t + 1) ** alpha)):
            break
    else:
        held += [(s / steps ** alpha, toks) for s, toks in live]
    return sorted(held, key=lambda h: -h[0])[:beams]
