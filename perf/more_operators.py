"""Operators of beam search over the paged cache, as cases that can be timed.

A batch holds G requests (groups) of W beams. Kinds:
- select:  logits [G W, V] and the beams' scores [G, W] become the k best
           continuations of every group: score + log-softmax over all beams
           and tokens, in falling order, equal ones by beam and then token
- advance: of those, the first W that do not end are the next beams; ended ones
           among the first W join the group's list of finished hypotheses
- reorder: the next beams' block tables and partly filled pages follow their
           parents, in a 16-bit or an 8-bit cache of several layers
- maps:    block tables and slot maps of packed rows from request lengths
- trace:   hypotheses read back from the logs of tokens and parents

A cache of 16 bits is K and V [layers, blocks, P, KV, D]. One of 8 bits is tiles
of 16 tokens, [layers, blocks, KV, P / 16, 16 * D] bytes for K and for V, and
[layers, blocks, KV, P / 16, 32] bytes of scale codes.
"""
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INF = float("inf")


def _select(name, groups, beams, vocab, k, mix, dtype="bf16", pad=0, banned=0.0, dead=0.0):
    """pad: columns behind a row of logits; banned: share of tokens at -inf; dead: of beams."""
    return {"name": name, "kind": "select", "groups": groups, "beams": beams, "vocab": vocab, "k": k,
            "mix": mix, "dtype": dtype, "pad": pad, "banned": banned, "dead": dead}


def _advance(name, groups, beams, k, steps, mix, ends=1, alpha=1.0, early=False):
    return {"name": name, "kind": "advance", "groups": groups, "beams": beams, "k": k, "steps": steps,
            "mix": mix, "ends": ends, "alpha": alpha, "early": early}


def _reorder(name, groups, beams, tokens, mix, layers=28, kv_heads=8, dim=128, page=16, cache="bf16"):
    return {"name": name, "kind": "reorder", "groups": groups, "beams": beams, "least": tokens[0],
            "most": tokens[1], "mix": mix, "layers": layers, "kv_heads": kv_heads, "dim": dim,
            "page": page, "cache": cache}


def _maps(name, requests, cached, new, mix, page=16):
    return {"name": name, "kind": "maps", "requests": requests, "cached_min": cached[0],
            "cached_max": cached[1], "new_min": new[0], "new_max": new[1], "mix": mix, "page": page}


def _trace(name, groups, beams, steps, mix):
    return {"name": name, "kind": "trace", "groups": groups, "beams": beams, "steps": steps, "mix": mix}


def listed():
    return [
        # a step of one request with four beams over a model's vocabulary: the smallest selection
        _select("select_c1", 1, 4, 151936, 8, 1),
        # wide beams on a served batch: the largest logits
        _select("select_wide", 32, 8, 151936, 16, 3),
        # a small odd vocabulary in 32 bits, rows inside a padded product, banned tokens, dead beams
        _select("select_odd", 5, 5, 32003, 15, 4, dtype="fp32", pad=29, banned=0.3, dead=0.2),
        # bookkeeping of one request's step
        _advance("advance_c1", 1, 4, 8, 128, 5),
        # of a full batch with two end tokens
        _advance("advance_c64", 64, 16, 48, 512, 6, ends=2, alpha=0.6, early=True),
        # the cache follows the beams of one request
        _reorder("reorder_c1", 1, 4, (300, 700), 7),
        # of a batch, all layers of a larger model
        _reorder("reorder_c16", 16, 4, (300, 4000), 8, layers=36),
        # the same from an 8-bit cache with wider pages and beams
        _reorder("reorder_8bit", 8, 8, (300, 4000), 9, layers=36, page=32, cache="8bit"),
        # metadata of a decode step: one new token for each of many long requests
        _maps("maps_decode", 64, (1024, 32000), (1, 1), 10),
        # of a block of packed prompts, some of them continued
        _maps("maps_prompts", 23, (0, 3000), (1, 700), 11),
        # one request's answers
        _trace("trace_c1", 1, 4, 100, 2),
        # the answers of a batch of long searches
        _trace("trace_long", 16, 8, 2048, 12),
    ]


def _log(rng, lo, hi):
    """An integer in [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("select", "select", "select", "advance", "reorder", "reorder", "maps", "trace"))
    mix = rng.randrange(1 << 20)
    beams = rng.choice((1, 2, 3, 4, 4, 5, 8, 16, 32))
    if kind == "select":
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        vocab = _log(rng, 500, 160000)
        groups = _log(rng, 1, max(1, min(64, 17000000 // (beams * vocab))))
        k = min(64, rng.choice((beams, 2 * beams, 2 * beams, 3 * beams)))
        return _select("", groups, beams, vocab, k, mix, dtype, pad=rng.choice((0, 0, 7, 64)),
                       banned=rng.choice((0.0, 0.0, 0.01, 0.5)), dead=rng.choice((0.0, 0.0, 0.3)))
    if kind == "advance":
        return _advance("", _log(rng, 1, 64), beams, min(64, beams * rng.choice((1, 2, 3))),
                        _log(rng, 8, 512), mix, ends=rng.choice((1, 1, 2)),
                        alpha=rng.choice((0.0, 0.6, 1.0)), early=rng.random() < 0.5)
    if kind == "reorder":
        least = _log(rng, 1, 2000)
        return _reorder("", _log(rng, 1, max(1, 64 // beams)), beams, (least, 2 * least), mix,
                        layers=rng.choice((2, 8, 28, 36)), kv_heads=rng.choice((8, 8, 4, 5)),
                        dim=rng.choice((128, 128, 64)), page=rng.choice((16, 16, 32, 64)),
                        cache=rng.choice(("bf16", "fp16", "8bit")))
    if kind == "maps":
        new = rng.choice((1, _log(rng, 2, 2000)))
        requests = _log(rng, 1, 64)
        return _maps("", requests, (0, _log(rng, 1, 32000)), (1, max(1, new // requests)), mix,
                     page=rng.choice((16, 16, 32, 64)))
    return _trace("", _log(rng, 1, 16), beams, _log(rng, 4, 2048), mix)


# ---- inputs ----------------------------------------------------------------------------------


def _lengths(case):
    """Of a reorder: cached tokens of every group. Of maps: cached and new tokens of every request."""
    rng = random.Random(case["mix"])
    if case["kind"] == "reorder":
        return [rng.randint(case["least"], case["most"]) for _ in range(case["groups"])]
    n = case["requests"]
    return ([rng.randint(case["cached_min"], case["cached_max"]) for _ in range(n)],
            [rng.randint(case["new_min"], case["new_max"]) for _ in range(n)])


def prepare(case, seed):
    gen = torch.Generator(DEV).manual_seed(seed * 1000003 + case["mix"])
    s = {"case": case}

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    def whole(lo, hi, *shape, dtype=torch.int32):
        """Integers in [lo, hi)."""
        return torch.randint(lo, hi, shape, device=DEV, generator=gen).to(dtype)

    def some(share, *shape):
        return torch.rand(*shape, device=DEV, generator=gen) < share

    if case["kind"] == "maps":
        cached, new = _lengths(case)
        P = case["page"]
        pages = [-(-(a + b) // P) for a, b in zip(cached, new)]
        s["lengths"] = torch.tensor([a + b for a, b in zip(cached, new)], dtype=torch.int32, device=DEV)
        s["starts"] = torch.tensor(cached, dtype=torch.int32, device=DEV)
        s["counts"] = torch.tensor(new, dtype=torch.int32, device=DEV)
        s["blocks"] = torch.randperm(sum(pages) + 9, device=DEV, generator=gen)[:sum(pages)].to(torch.int32)
        s["width"], s["rows"] = max(pages) + 3, sum(new)
        return s

    G, W = case["groups"], case["beams"]
    if case["kind"] == "select":
        V = case["vocab"]
        # next-token logits: a broad spread, a few tokens far above it, another level per row
        x = normal(G * W, V + case["pad"]).mul_(2.0).add_(normal(G * W, 1))
        top = whole(0, V, G * W, 12, dtype=torch.int64)
        x.scatter_add_(1, top, 6.0 + 3.0 * normal(G * W, 12))
        x[some(case["banned"], G * W, V + case["pad"])] = -INF
        s["logits"] = x.to(DTYPES[case["dtype"]])[:, :V]
        scores = (-20.0 * torch.rand(G, W, device=DEV, generator=gen)).sort(-1, descending=True)[0]
        s["scores"] = scores.masked_fill(some(case["dead"], G, W), -INF)
        return s
    if case["kind"] == "advance":
        T, K = case["steps"], case["k"]
        token = whole(10, 30000, G, K, dtype=torch.int64)
        end = some(0.25, G, K)                              # long answers: many candidates end
        s["ends"] = torch.tensor([3, 7][:case["ends"]], device=DEV)
        token = torch.where(end, s["ends"][whole(0, case["ends"], G, K, dtype=torch.int64)], token)
        score = (-20.0 - 10.0 * torch.rand(G, K, device=DEV, generator=gen)).sort(-1, descending=True)[0]
        s["candidates"] = {"score": score, "beam": whole(0, W, G, K), "token": token}
        length = whole(1, T, G)
        held = torch.arange(W, device=DEV) < whole(0, W + 1, G, 1)      # finished so far
        old = (-1.5 - 2.0 * torch.rand(G, W, device=DEV, generator=gen)).sort(-1, descending=True)[0]
        s["state"] = {
            "scores": (-20.0 * torch.rand(G, W, device=DEV, generator=gen)).sort(-1, descending=True)[0],
            "length": length, "done": some(0.1, G).int(),
            "ids": whole(10, 30000, G, W, dtype=torch.int64),
            "position": (100 + length)[:, None].repeat(1, W),
            "parents": whole(0, W, G, W), "token_log": whole(0, 30000, T, G, W),
            "parent_log": whole(0, W, T, G, W),
            "fin_scores": old.masked_fill(~held, -INF),
            "fin_length": whole(1, T, G, W).masked_fill(~held, 0),
            "fin_beam": whole(0, W, G, W).masked_fill(~held, 0),
            "fin_token": whole(0, 9, G, W).masked_fill(~held, 0)}
        # (the next state goes into buffers of its own; the logs are one for all steps)
        s["out"] = {k: v if k.endswith("_log") else torch.empty_like(v) for k, v in s["state"].items()}
        return s
    if case["kind"] == "trace":
        T = case["steps"]
        # the parent of a beam is mostly a beam near the top
        s["parents"] = torch.minimum(whole(0, W, T, G, W), whole(0, W, T, G, W))
        s["tokens"] = whole(0, 150000, T, G, W)
        s["steps"], s["beams"] = whole(0, T + 1, G, W), whole(0, W, G, W)
        return s

    # reorder: a group's beams share the prompt's full pages and have pages of their own behind
    L, KV, D, P = case["layers"], case["kv_heads"], case["dim"], case["page"]
    lens = _lengths(case)
    shared = 40                                              # prompts' blocks, met again and again
    width = max(n // P for n in lens) + 2
    tables = whole(0, shared, G, 1, width).repeat(1, W, 1)
    at = torch.tensor([n // P for n in lens], device=DEV)[:, None, None] + torch.arange(2, device=DEV)
    private = torch.randperm(2 * G * W, device=DEV, generator=gen).to(torch.int32).view(G, W, 2) + shared
    tables.scatter_(2, at.expand(G, W, 2).clamp_max(width - 1), private)
    blocks = shared + 2 * G * W
    s["tables"] = tables.view(G * W, width).contiguous()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)[:, None].repeat(1, W)
    # as a search picks them: beams near the top have several children
    s["parents"] = torch.minimum(whole(0, W, G, W), whole(0, W, G, W))
    if case["cache"] == "8bit":
        def pool(n):
            return torch.randint(0, 120, (L, blocks, KV, P // 16, n), dtype=torch.uint8, device=DEV, generator=gen)
        s["pools"] = [pool(16 * D), pool(16 * D), pool(32)]
    else:
        s["pools"] = [normal(L, blocks, P, KV, D).to(DTYPES[case["cache"]]) for _ in range(2)]
    return s


# ---- the plain forms -------------------------------------------------------------------------


def _best(s):
    """Scores differ by less than 32 bits hold where the choice is close: in 64."""
    c, score = s["case"], s["scores"].double()
    G, W = score.shape
    x = s["logits"].double().view(G, W, -1)
    alive = score > -INF
    broken = alive & ~(x < INF).all(-1)
    m = x.masked_fill(~(x < INF), 0.0).amax(-1, keepdim=True).clamp_min(-1e300)
    total = torch.log(torch.exp(x - m).sum(-1, keepdim=True)) + m
    live = alive & ~broken & (total[..., 0] > -INF)
    x = torch.where(live[..., None], score[..., None] + x - total, -INF)
    value, place = torch.sort(x.view(G, -1), dim=-1, descending=True, stable=True)
    place = place[:, :c["k"]]
    V = c["vocab"]
    return [value[:, :c["k"]].float(), (place // V).int(), place % V, broken.view(-1).int()]


def _next(s):
    c, cand, old, new = s["case"], s["candidates"], s["state"], s["out"]
    G, W = old["scores"].shape
    T, K = c["steps"], c["k"]
    own_beam = torch.arange(W, device=DEV, dtype=torch.int32).expand(G, W)
    t = old["length"]
    runs = (old["done"] == 0) & (t < T)
    valid = cand["score"] > -INF
    ends = valid & (cand["token"][..., None] == s["ends"]).any(-1)
    goes = valid & ~ends

    # the n-th candidate that goes on, for n < W
    hit = goes[:, None] & (goes.cumsum(-1)[:, None] == own_beam[..., None] + 1)       # [G, W, K]
    found, at = hit.any(-1), hit.int().argmax(-1)
    live = runs[:, None]

    def pick(x, otherwise, done):
        return torch.where(live, torch.where(found, x.gather(1, at), otherwise), done)

    zero = torch.zeros_like(old["ids"])
    parents = pick(cand["beam"], own_beam, own_beam)
    ids = pick(cand["token"], zero, zero)
    scores = pick(cand["score"], torch.full_like(old["scores"], -INF), old["scores"])

    # finished: the best W of those there were and those that end now, older ones first
    power = (t + 1).double()[:, None] ** c["alpha"]
    take = ends & (torch.arange(K, device=DEV) < W) & live
    fresh = torch.where(take, cand["score"].double() / power, -INF).float()
    fin = torch.cat([old["fin_scores"], fresh], 1)
    order = torch.sort(fin, dim=-1, descending=True, stable=True)[1][:, :W]

    def keep(name, x):
        both = torch.cat([old[name], torch.where(take, x, 0).int()], 1)
        return both.gather(1, order)

    fin_length = keep("fin_length", (t + 1)[:, None])
    fin_scores = fin.gather(1, order)
    best = (scores[:, 0].double() / power[:, 0]).float()
    enough = (fin_length[:, -1] > 0) & (c["early"] | (fin_scores[:, -1] >= best))
    stop = (scores[:, 0] == -INF) | enough | (t + 1 >= T)
    result = {
        "scores": scores, "length": t + runs, "done": torch.where(runs, stop.int(), old["done"]),
        "ids": ids, "position": old["position"] + live, "parents": parents,
        "fin_scores": fin_scores, "fin_length": fin_length,
        "fin_beam": keep("fin_beam", cand["beam"]), "fin_token": keep("fin_token", cand["token"])}
    for name, x in result.items():
        new[name].copy_(x)
    step, group = t.long().clamp_max(T - 1), torch.arange(G, device=DEV)
    for name, x in (("token_log", ids), ("parent_log", parents)):
        log = new[name]
        log[step, group] = torch.where(live, x.int(), log[step, group])
    return new


def _children(parents, page):
    """For every next beam the page it takes over of `page` [G, W], and the one it continues."""
    W = parents.shape[1]
    p = parents.long()
    beam = torch.arange(W, device=DEV)
    same = p[:, :, None] == p[:, None, :]
    first = ~(same & (beam[None, :] < beam[:, None])).any(-1)
    childless = ~(p[:, :, None] == beam).any(1)
    # the r-th beam that is not the first child takes the page of the r-th without children
    further = (~first).cumsum(-1) * ~first
    spare = childless.cumsum(-1) * childless
    match = (further[:, :, None] == spare[:, None, :]) & ~first[:, :, None] & childless[:, None, :]
    source = page.gather(1, p)
    return torch.where(first, source, page.gather(1, match.int().argmax(-1))), source


def _follow(s):
    c = s["case"]
    G, W, P = c["groups"], c["beams"], c["page"]
    n = s["lens"][:, :1].long()
    tables = s["tables"].view(G, W, -1)
    column = torch.arange(tables.shape[2], device=DEV)
    at = n // P
    page = tables.gather(2, at[:, None].expand(G, W, 1))[..., 0]
    taken, source = _children(s["parents"], page)
    taken = torch.where(n % P > 0, taken, page)
    moved = tables.gather(1, s["parents"].long()[..., None].expand_as(tables))
    moved = torch.where(column < at[..., None], moved, tables)
    moved = torch.where(column == at[..., None], taken[..., None], moved)
    tables.copy_(moved)
    fill = (n % P).expand(G, W).reshape(-1)
    to, from_ = taken.reshape(-1).long(), torch.where(n % P > 0, source, page).reshape(-1).long()
    if c["cache"] == "8bit":
        keep = torch.arange(P // 16, device=DEV) * 16 < fill[:, None]                 # [G W, P / 16]
        keep = keep[:, None, :, None]
    else:
        keep = (torch.arange(P, device=DEV) < fill[:, None])[:, :, None, None]
    for pool in s["pools"]:
        pool[:, to] = torch.where(keep, pool[:, from_], pool[:, to])
    return [s["tables"]] + s["pools"]


def _map(s):
    P, W, R = s["case"]["page"], s["width"], s["rows"]
    pages = (s["lengths"].long() + P - 1) // P
    j = torch.arange(W, device=DEV)
    at = (pages.cumsum(0) - pages)[:, None] + j
    tables = torch.where(j < pages[:, None], s["blocks"][at.clamp_max(len(s["blocks"]) - 1)], 0)
    end = s["counts"].long().cumsum(0)
    first = end - s["counts"]
    row = torch.arange(R, device=DEV)
    seq = (row[:, None] >= end).sum(-1)
    position = s["starts"][seq].long() + row - first[seq]
    return [tables, seq.int(), position, tables[seq, position // P].long(), position % P,
            (position + 1).int(), first.int()]


def _walk(s):
    """Every step's beam at once: jumps of 1, 2, 4 ... steps back, as the distance's bits want."""
    T, G, W = s["parents"].shape
    t = torch.arange(T, device=DEV)
    steps = s["steps"].long()
    left = (steps[..., None] - 1 - t).clamp_min(0)                                    # [G, W, T]
    step = (steps[..., None] - 1).expand(G, W, T).clamp_min(0)
    beam = s["beams"].long()[..., None].expand(G, W, T)
    group = torch.arange(G, device=DEV)[:, None, None]
    jump = s["parents"].long()                                                        # 2 ** i back
    for i in range(max(1, (T - 1).bit_length())):
        hop = (left >> i & 1) == 1
        beam = torch.where(hop, jump[step, group, beam], beam)
        step = step - (hop.long() << i)
        before = (t - (1 << i)).clamp_min(0)
        jump = jump[before].gather(2, jump)
    inside = t < steps[..., None]
    return torch.where(inside, s["tokens"][t, group, beam].long(), -1)


def _plain(s):
    kind = s["case"]["kind"]
    return {"select": _best, "advance": _next, "reorder": _follow, "maps": _map, "trace": _walk}[kind](s)


# ---- the framework's -------------------------------------------------------------------------


def _own(s):
    from acorninfer_amd.ops import beam, request_maps
    c = s["case"]
    kind = c["kind"]
    if kind == "select":
        return list(beam.beam_select(s["logits"], s["scores"], c["k"]))
    if kind == "advance":
        cand = s["candidates"]
        out = beam.beam_advance(beam.BeamState(**s["state"]), beam.BeamCandidates(**cand), s["ends"],
                                length_penalty=c["alpha"], early_stopping=c["early"],
                                out=beam.BeamState(**s["out"]))
        return out._asdict()
    if kind == "reorder":
        k, v, *scales = s["pools"]
        beam.beam_reorder(k, v, s["tables"], s["lens"], s["parents"],
                          scale_pool=scales[0] if scales else None)
        return [s["tables"]] + s["pools"]
    if kind == "trace":
        return beam.beam_trace(s["tokens"], s["parents"], s["steps"], s["beams"], pad=-1)
    tables = request_maps.block_tables(s["blocks"], s["lengths"], c["page"], s["width"])
    return [tables] + list(request_maps.slot_map(tables, s["starts"], s["counts"], c["page"], s["rows"]))


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    kind = case["kind"]
    if kind == "maps":
        cached, new = _lengths(case)
        P, n, R = case["page"], case["requests"], sum(new)
        pages = [-(-(a + b) // P) for a, b in zip(cached, new)]
        moved = 4 * (sum(pages) + n * (max(pages) + 3) + 4 * n) + R * (4 + 4 + 8 + 8 + 8 + 4)
        return {"bytes": moved, "flops": 4 * (R + sum(pages))}
    G, W = case["groups"], case["beams"]
    if kind == "select":
        size = DTYPES[case["dtype"]].itemsize
        n = G * W * case["vocab"] * (1 - case["dead"])
        return {"bytes": n * size + G * (W * 8 + case["k"] * 16), "flops": 5 * n}
    if kind == "advance":
        return {"bytes": G * (case["k"] * 16 + W * 80 + 16), "flops": 4 * G * case["k"]}
    if kind == "trace":
        n = G * W * case["steps"]
        return {"bytes": n * (4 + 4 + 4), "flops": n}
    lens, P, D = _lengths(case), case["page"], case["dim"]
    size, filled = 2, [n % P for n in lens]
    if case["cache"] == "8bit":                              # whole tiles, with their scale codes
        size, filled = 1 + 1 / D, [-(-n // 16) * 16 for n in filled]
    # with parents as prepare() draws them (the smaller of two) this share of beams needs a copy
    copies = sum((1 - ((W - b) ** 2 - (W - b - 1) ** 2) / W ** 2) ** W for b in range(W)) / W
    token = case["layers"] * 2 * case["kv_heads"] * D * size
    table = 8 * W * sum(n // P for n in lens)
    return {"bytes": 2 * copies * W * sum(filled) * token + table, "flops": W * sum(n // P for n in lens)}


# ---- in 64 bits ------------------------------------------------------------------------------


def _exact_best(s):
    c = s["case"]
    V, k = c["vocab"], c["k"]
    value, beam, token, status = [], [], [], []
    for x, score in zip(s["logits"].view(c["groups"], c["beams"], V), s["scores"]):
        y = torch.log_softmax(x.double(), -1) + score.double()[:, None]
        bad = torch.isnan(x).any(-1) | (x == INF).any(-1)
        gone = bad | (score == -INF) | (x == -INF).all(-1)
        y[gone] = -INF
        flat = y.view(-1)
        at = torch.nonzero(flat >= torch.kthvalue(flat, flat.numel() - k + 1)[0])[:, 0]
        v, order = torch.sort(flat[at], descending=True, stable=True)
        at = at[order[:k]]
        value.append(v[:k])
        beam.append((at // V).int())
        token.append(at % V)
        status.append((bad & (score > -INF)).int())
    return [torch.stack(value), torch.stack(beam), torch.stack(token), torch.cat(status)]


def _exact_next(s):
    c = s["case"]
    G, W, T = c["groups"], c["beams"], c["steps"]
    st = {k: v.tolist() for k, v in s["state"].items() if not k.endswith("_log")}
    cand = {k: v.tolist() for k, v in s["candidates"].items()}
    ends = s["ends"].tolist()
    logs = {k: s["state"][k].clone() for k in ("token_log", "parent_log")}
    for g in range(G):
        t = st["length"][g]
        st["parents"][g], st["ids"][g], score = list(range(W)), [0] * W, [-INF] * W
        if st["done"][g] or t >= T:
            continue
        n = 0
        held = [e for e in zip(*(st[k][g] for k in ("fin_scores", "fin_length", "fin_beam", "fin_token")))
                if e[1]]
        for i in range(c["k"]):
            v, b, token = (cand[k][g][i] for k in ("score", "beam", "token"))
            if not v > -INF:
                continue
            if token in ends:
                if i < W:
                    held.append((v / (t + 1) ** c["alpha"], t + 1, b, token))
            elif n < W:
                st["parents"][g][n], st["ids"][g][n], score[n] = b, token, v
                n += 1
        held = sorted(held, key=lambda e: -e[0])[:W]
        full = len(held) == W
        st["scores"][g], st["length"][g] = score, t + 1
        st["position"][g] = [x + 1 for x in st["position"][g]]
        st["done"][g] = int(n == 0 or t + 1 >= T or full and (
            c["early"] or held[-1][0] >= score[0] / (t + 1) ** c["alpha"]))
        held += [(-INF, 0, 0, 0)] * (W - len(held))
        for k, column in zip(("fin_scores", "fin_length", "fin_beam", "fin_token"), zip(*held)):
            st[k][g] = list(column)
        logs["token_log"][t, g] = torch.tensor(st["ids"][g], dtype=torch.int32, device=DEV)
        logs["parent_log"][t, g] = torch.tensor(st["parents"][g], dtype=torch.int32, device=DEV)
    return {k: logs[k] if k in logs else torch.tensor(
        st[k], dtype=torch.float64 if v.dtype.is_floating_point else v.dtype) for k, v in s["state"].items()}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "select":
        return _exact_best(s)
    if case["kind"] == "advance":
        return _exact_next(s)
    return None                                              # whole numbers and copies: no rounding
