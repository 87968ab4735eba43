"""Beam search over a paged cache: one pass of an operator on one GPU.

Kinds of a case: `select` (the best continuations of every request's beams), `fork` (children inherit their parents' pages or state
slots, and what they cannot share is copied), `tables` (page lists, positions and slots of a step from tables and lengths) and `attend`
(attention of one token of every beam, over pages of which a request's beams share the first ones).

    select  value of token v behind beam b: score_b + z_v - log sum_u exp z_u; what is no number counts as -inf.  The n largest of a
            request, ties to the lowest (b, v); where there is no candidate above -inf: parent and token -1.  `next`: the first ones of
            them whose token does not end a sequence, as many as there are beams.
    fork    a child takes the full pages of its parent's table; a page that is partly filled goes to the parent's first child, the others
            have it copied into a fresh page; where all pages are full, a fresh one is added.  Fresh pages are the first ones
            of the request's own pages that no child has kept, one after the other.  A row behind its last page: -1.  A child without a
            parent is a dead row: length -1.
    tables  of rows with `cached` tokens and `counts` new ones: pages one row after the other, where each row's begin, tokens on the last
            page, and of every new token position and slot (page x page size + offset).  Behind the last: 0, and slot -1.
            A row that sits the step out has no pages.  `shared`: how many full pages at the beginning the rows of a request have in common.
"""
import math
import random

import torch

own = False
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


# ---------------------------------------------------------------------------------------------------------- cases
def _select(name, requests, beams, vocab, *, n=0, ended=1, masked=0.0, dead=0.0, dtype="bfloat16"):
    return {"name": name, "kind": "select", "requests": requests, "beams": beams, "vocab": vocab, "n": n or 2 * beams, "ended": ended,
            "masked": masked, "dead": dead, "dtype": dtype}


def _pages(name, kind, requests, beams, prompt, new, *, layers=1, heads=(32, 8), dim=128, page=64, ragged=False, cap=0.0, sink=False,
           what="pages", rows=0, dead=0.0, dtype="bfloat16"):
    """`prompt`: tokens of all prompts; `new`: tokens that every beam has behind its prompt; `rows`: of a step of portions, new tokens of all rows"""
    return {"name": name, "kind": kind, "requests": requests, "beams": beams, "prompt": prompt, "new": new, "layers": layers, "q_heads": heads[0],
            "kv_heads": heads[1], "dim": dim, "page": page, "ragged": ragged, "cap": cap, "sink": sink, "what": what, "rows": rows, "dead": dead,
            "dtype": dtype}


def listed():
    return [
        # one user's request with four beams
        _select("select 1 x 4", 1, 4, 128256),
        # the largest decode batch, eight beams each, two tokens that end a sequence
        _select("select 32 x 8", 32, 8, 128256, n=24, ended=2),
        # logits in 32 bits, an odd vocabulary, tokens that a grammar hides, beams that have ended
        _select("select 13 x 5 masked", 13, 5, 50257, masked=0.9, dead=0.2, dtype="float32"),
        # one user's request: four beams of 8 layers part ways
        _pages("fork 1 x 4", "fork", 1, 4, 977, 37, layers=8),
        # the largest decode batch
        _pages("fork 32 x 8", "fork", 32, 8, 32 * 150, 45, layers=8, ragged=True),
        # state slots of recurrent layers, copied whole
        _pages("fork states 12 x 5", "fork", 12, 5, 12, 0, layers=6, heads=(16, 16), what="states", dtype="float32"),
        # tables of one user's request
        _pages("tables 1 x 4", "tables", 1, 4, 977, 37),
        # portions of prompts and single tokens in one step, small pages
        _pages("tables 61 portions", "tables", 61, 1, 61 * 900, 0, page=16, ragged=True, rows=8192),
        # one user's request, token by token: latency
        _pages("attend 1 x 4", "attend", 1, 4, 977, 37),
        # one long document, four beams
        _pages("attend 1 x 4 long", "attend", 1, 4, 100003, 141),
        # the largest decode batch: prompts of very different lengths
        _pages("attend 32 x 8", "attend", 32, 8, 32 * 1200, 101, ragged=True, dead=0.05),
        # small heads and pages, a soft cap and a sink, the second 16-bit type
        _pages("attend 7 x 5 small heads", "attend", 7, 5, 7 * 1500, 61, heads=(16, 4), dim=64, page=16, ragged=True, cap=50.0, sink=True, dtype="float16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["select", "select", "fork", "fork", "tables", "attend", "attend", "attend"])
    beams = rng.choice([1, 2, 3, 4, 4, 5, 6, 8, 8, 10, 16])
    requests = _log(rng, 1, 256 // beams)
    if kind == "select":
        case = _select("", requests, beams, _log(rng, 40, 152064) if rng.random() < 0.5 else rng.choice([32000, 50257, 50272, 128256, 131072]),
                       n=rng.choice([1, 2, 3]) * beams, ended=rng.choice([0, 1, 2]), masked=rng.choice([0.0, 0.0, 0.5, 0.99]),
                       dead=rng.choice([0.0, 0.3]), dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]))
        case["requests"] = max(1, min(requests, 128256 * 256 // (case["vocab"] * beams * (2 if case["dtype"] == "float32" else 1))))
        del case["name"]
        return case
    kv = rng.choice([1, 2, 4, 8, 8])
    dim = rng.choice([128, 128, 64])
    more = dict(heads=(kv * rng.choice([1, 2, 4, 4, 5, 8]), kv), dim=dim, page=rng.choice([16, 64, 64, 128]), ragged=rng.random() < 0.7,
                dead=rng.choice([0.0, 0.0, 0.2]), dtype=rng.choice(["bfloat16", "bfloat16", "float16"]))
    new = rng.choice([0, 1, _log(rng, 1, 300), _log(rng, 1, 300)])
    if kind == "attend":
        if rng.random() < 0.3:
            more.update(cap=50.0)
        if rng.random() < 0.3:
            more.update(sink=True)
        case = _pages("", kind, requests, beams, requests * _log(rng, 1, max(1, min(100000, 80000 // (requests * beams)))), new, **more)
    elif kind == "tables":
        prompt = requests * _log(rng, 1, max(1, min(100000, 400000 // requests)))
        if rng.random() < 0.5:
            case = _pages("", kind, requests, beams, prompt, new, **more)
        else:
            case = _pages("", kind, requests, 1, prompt, 0, rows=max(requests, _log(rng, 1, 8192)), **more)
    else:
        what = rng.choice(["pages", "pages", "quantised", "states"])
        more["layers"] = rng.choice([1, 2, 4, 8]) if more["page"] < 128 else rng.choice([1, 2, 4])
        if what == "states":
            requests = min(requests, 60 // beams)
            case = _pages("", kind, requests, beams, requests, 0, what=what, **dict(more, dtype="float32"))
        else:
            case = _pages("", kind, requests, beams, requests * _log(rng, 1, 150), min(new, 60), what=what, **more)
    del case["name"]
    return case


def _spread(case, total):
    """`total` over the requests, one at least for each: equal, or spread over a factor of sixteen.  A matter of the case alone."""
    n = case["requests"]
    rng = random.Random(n * 1000003 + total)
    w = [math.exp(rng.uniform(0.0, math.log(16.0))) if case["ragged"] else 1.0 for _ in range(n)]
    out = [max(1, int(total * x / sum(w))) for x in w]
    while sum(out) != total:
        i = rng.randrange(n)
        out[i] += 1 if sum(out) < total else -1 if out[i] > 1 else 0
    return out


def _shape(case):
    """What a pass looks like, a matter of the case alone: per row the tokens in the cache (-1: dead) and the pages by number; the new tokens of each
    row (portions), the pages that each request owns, and how many there are.  Beams share their prompt's full pages."""
    rng = random.Random(7)
    k, page = case["beams"], 2 if case["what"] == "states" else case["page"]
    cached, tables, owned, total = [], [], [], 0
    for n in _spread(case, case["prompt"]):
        live = [rng.random() >= case["dead"] for _ in range(k)]
        live[0] = True
        length, first = n + case["new"], total
        common = n // page
        for b in range(k):
            cached.append(length if live[b] else -1)
            mine = -(-length // page) - common
            tables.append(list(range(first, first + common)) + list(range(total + common, total + common + mine)) if live[b] else [])
            total += mine
        total += common
        spare = k * (1 + -(-length // page) - common)
        owned.append((first, total, spare))
        total += spare
    counts = [1] * len(cached)
    if case["rows"]:
        counts = _spread(case, case["rows"])
        rng.shuffle(counts)
    return cached, tables, owned, counts, total


def _parents(case, cached):
    """Which beam each child of a request comes from: often the first ones."""
    rng, k, out = random.Random(11), case["beams"], []
    for q in range(case["requests"]):
        live = [b for b in range(k) if cached[q * k + b] >= 0]
        out.append([rng.choice(live[:1 + rng.randrange(len(live))]) for _ in range(k)])
        if rng.random() < case["dead"]:
            out[-1][-1] = -1
    return out


# ---------------------------------------------------------------------------------------------------------- inputs
def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _padded(rows, width):
    return _int32([r + [-1] * (width - len(r)) for r in rows])


def _select_inputs(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    Q, k, V = case["requests"], case["beams"], case["vocab"]
    # as models have them: most tokens unlikely, a few that stand out
    logits = torch.randn(Q * k, V, generator=gen, device="cuda").mul_(2.0)
    at = torch.randint(0, V, (Q * k, 12), generator=gen, device="cuda")
    logits.scatter_add_(1, at, 8.0 + 2.0 * torch.randn(Q * k, 12, generator=gen, device="cuda"))
    if case["masked"]:
        logits.masked_fill_(torch.rand(1, V, generator=gen, device="cuda") < case["masked"], -math.inf)
    scores = -20.0 * torch.rand(Q * k, generator=gen, device="cuda")
    if case["dead"]:
        scores.masked_fill_(torch.rand(Q * k, generator=gen, device="cuda") < case["dead"], -math.inf)
    ended = torch.randint(0, V, (case["ended"],), generator=gen, device="cuda").to(torch.int32)
    ended[:1] = at[0, 0].to(torch.int32)      # (one that a beam may well take)
    return {"case": case, "logits": logits.to(DTYPES[case["dtype"]]), "scores": scores, "ended": ended}


def prepare(case, seed):
    if case["kind"] == "select":
        return _select_inputs(case, seed)
    gen = torch.Generator("cuda").manual_seed(seed)
    H, D, page, dt = case["kv_heads"], case["dim"], case["page"], DTYPES[case["dtype"]]
    cached, tables, owned, counts, total = _shape(case)
    place = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()      # pages, as a pool hands them out
    tables = [[place[p] for p in t] for t in tables]
    state = {"case": case, "cached": _int32(cached), "num_pages": total + 1}
    width = max(len(t) for t in tables) + 1
    if case["kind"] == "fork":
        state["table"], state["parents"] = _padded(tables, width), _int32(_parents(case, cached))
        pages = [[place[p] for p in range(a, b + n)] for a, b, n in owned]
        most = max(len(p) for p in pages)
        state["pool"] = _padded(pages, most)
        shape, L = (total + 1, 2, page, H, D), case["layers"]
        if case["what"] == "quantised":
            # (bytes of pages in 4 bits: codes, scales; what they say does not matter here)
            state["cache"] = torch.randint(0, 256, (L, total + 1, H, page // 16, 16 * (D + 8 * (D // 32))), generator=gen, device="cuda", dtype=torch.uint8)
        elif case["what"] == "states":
            state["cache"] = torch.randn(L, total + 1, H, D, D, generator=gen, device="cuda")
        else:
            state["cache"] = torch.empty(L, *shape, dtype=dt, device="cuda").normal_(generator=gen)
        return state
    if case["rows"]:        # (the row's pages for its new tokens too)
        more = total
        for i, (n, c) in enumerate(zip(counts, cached)):
            need = -(-(c + n) // page)
            tables[i] += range(more, more + need - len(tables[i]))
            more = max([more, *(p + 1 for p in tables[i])])
        width = max(len(t) for t in tables)
        state["num_pages"] = more
    if case["kind"] == "tables":
        if not case["rows"]:
            tables = [t + [total] if c >= 0 and c % page == 0 else t for t, c in zip(tables, cached)]
        state["table"], state["counts"] = _padded(tables, width), _int32(counts) if case["rows"] else None
        state["tokens"] = sum(counts)
        return state
    R = len(cached)
    start = torch.tensor([0, *(len(t) for t in tables)]).cumsum(0)
    state.update(indices=_int32([p for t in tables for p in t]), indptr=start.to(torch.int32).cuda(),
                 last=_int32([(n - 1) % page + 1 if n > 0 else 0 for n in cached]),
                 shared=_int32([n // page for n in _spread(case, case["prompt"])]), longest=max(cached))
    state["kv"] = torch.empty(total + 1, 2, page, H, D, dtype=dt, device="cuda").normal_(generator=gen)
    q = torch.zeros(R, (case["q_heads"] + 2 * H) * D, dtype=dt, device="cuda")
    q[:, :case["q_heads"] * D].normal_(generator=gen)
    state.update(q=q, sink=torch.randn(case["q_heads"], generator=gen, device="cuda").to(dt) if case["sink"] else None)
    if own:
        # what a serving process keeps: scratch
        from blitz_scale_b200 import ops
        n = ops.attn_beams_workspace_bytes(R, case["beams"], q_heads=case["q_heads"], kv_heads=H, head_dim=D, device="cuda")
        state["scratch"] = torch.zeros(n, dtype=torch.uint8, device="cuda")
    return state


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_select(state):
    case = state["case"]
    Q, k, n = case["requests"], case["beams"], case["n"]
    z = state["logits"].double()       # (a candidate near another one's value has to stay on its side)
    top = z.amax(1, keepdim=True)
    v = state["scores"].double()[:, None] + (z - (top + torch.exp(z - top).sum(1, keepdim=True).log()))
    v = torch.where(torch.isnan(v), -math.inf, v).view(Q, -1)
    v, at = torch.sort(v, dim=1, descending=True, stable=True)
    v, at = v[:, :n], at[:, :n]
    none = v == -math.inf
    parent, token = (torch.where(none, -1, t).to(torch.int32) for t in (at // case["vocab"], at % case["vocab"]))
    score = v.float()
    goes_on = ~none & (token[:, :, None] != state["ended"]).all(-1)
    first = torch.sort((~goes_on).to(torch.int8), dim=1, stable=True).indices[:, :k]       # those that go on, in their order
    real = goes_on.gather(1, first)
    return {"score": score, "parent": parent, "token": token, "next_score": torch.where(real, score.gather(1, first), -math.inf),
            "next_parent": torch.where(real, parent.gather(1, first), -1), "next_token": torch.where(real, token.gather(1, first), -1)}


def _plain_fork(state):
    case, table, pool = state["case"], state["table"], state["pool"]
    Q, k, W = case["requests"], case["beams"], table.shape[1]
    page = 2 if case["what"] == "states" else case["page"]
    old, P = table.view(Q, k, W).long(), state["num_pages"]
    par = state["parents"].long()
    cached = torch.where(par >= 0, state["cached"].view(Q, k).long().gather(1, par.clamp(min=0)), -1)
    alive, full, part = cached >= 0, cached.clamp(min=0) // page, cached.clamp(min=0) % page
    old = old.gather(1, par.clamp(min=0)[:, :, None].expand(-1, -1, W))
    again = ((par[:, :, None] == par[:, None, :]) & alive[:, None, :]).tril(-1).any(-1)      # an earlier child has the same parent
    keeps = full + ((part > 0) & ~again)
    i = torch.arange(W, device="cuda")
    kept = (i < keeps[:, :, None]) & alive[:, :, None]
    used = torch.zeros(Q, P + 1, dtype=torch.int32, device="cuda")
    used.scatter_(1, torch.where(kept, old, P).flatten(1), 1)
    free = (pool >= 0) & (used.gather(1, pool.clamp(min=0).long()) == 0)
    order = torch.sort((~free).to(torch.int8), dim=1, stable=True).indices
    fresh = pool.long().gather(1, order)
    needs = alive & ((part == 0) | again)
    mine = fresh.gather(1, (needs.cumsum(1) - 1).clamp(min=0))
    new = torch.where(kept, old, -1)
    new = torch.where((i == full[:, :, None]) & needs[:, :, None], mine[:, :, None], new)
    copies = needs & (part > 0)
    src = torch.where(copies, old.gather(2, full.clamp(max=W - 1)[:, :, None])[:, :, 0], -1).flatten()
    dst = torch.where(copies, mine, -1).flatten()
    tokens = torch.where(copies, part, 0).flatten()
    # the copies: a pair without one copies the last page, which nobody has, onto itself
    a, b, cache = torch.where(src >= 0, src, P - 1), torch.where(dst >= 0, dst, P - 1), state["cache"]
    if case["what"] == "pages":
        there = torch.arange(page, device="cuda") < tokens[:, None]
        cache[:, b] = torch.where(there[None, :, None, :, None, None], cache[:, a], cache[:, b])
    else:
        cache[:, b] = cache[:, a]
    to = lambda t: t.to(torch.int32)  # noqa: E731
    return {"table": to(new).view(Q * k, W), "cached": to(cached).flatten(), "src": to(src), "dst": to(dst), "tokens": to(tokens), "cache": cache}


def _plain_tables(state):
    case, table, page = state["case"], state["table"].long(), state["case"]["page"]
    R, W = table.shape
    cached = state["cached"].long()
    counts = state["counts"].long() if case["rows"] else (cached >= 0).long()
    length = torch.where(counts > 0, cached + counts, 0)
    pages = (length + page - 1) // page
    end, tok_end = pages.cumsum(0), counts.cumsum(0)
    zero = torch.zeros(1, dtype=torch.long, device="cuda")
    indptr, tok = torch.cat([zero, end]), torch.cat([zero, tok_end])
    e = torch.arange(R * W, device="cuda")
    row = torch.searchsorted(end, e, right=True).clamp(max=R - 1)
    indices = torch.where(e < end[-1], table.flatten()[(row * W + e - indptr[row]).clamp(0, R * W - 1)], 0)
    last = torch.where(pages > 0, length - (pages - 1) * page, 0)
    if case["rows"]:
        t = torch.arange(state["tokens"], device="cuda")
        of = torch.searchsorted(tok_end, t, right=True).clamp(max=R - 1)
        real, pos = t < tok_end[-1], cached[of] + t - tok[of]
    else:
        of = torch.arange(R, device="cuda")
        real, pos = cached >= 0, cached
    slot = torch.where(real, table[of, (pos // page).clamp(0, W - 1)] * page + pos % page, -1)
    pos = torch.where(real, pos, 0)
    out = {"indices": indices, "indptr": indptr, "last": last, "pos": pos, "slot": slot}
    if case["rows"]:
        out["tok_indptr"] = tok
    else:
        k = case["beams"]
        live, g = (length > 0).view(-1, k), table.view(-1, k, W)
        first = g.gather(1, live.to(torch.int8).argmax(1)[:, None, None].expand(-1, -1, W))       # of the first live row
        full = torch.where(live, length.view(-1, k) // page, W).amin(1)
        same = ((g == first) | ~live[:, :, None]).all(1).long().cumprod(1).sum(1)
        out["shared"] = torch.where(live.any(1), torch.minimum(full, same), 0)
    return {n: x.to(torch.int32) for n, x in out.items()}


def _plain_attend(state):
    case = state["case"]
    H, D, N, page = case["kv_heads"], case["dim"], case["q_heads"], case["page"]
    R = state["q"].shape[0]
    most = -(-state["longest"] // page)
    at = (state["indptr"][:-1, None] + torch.arange(most, device="cuda")).clamp(max=state["indices"].numel() - 1)
    kv = state["kv"][state["indices"][at].long()]                                             # [rows, pages, 2, page, heads, dim]
    k, v = (kv[:, :, i].reshape(R, most * page, H, D).float() for i in (0, 1))
    q = state["q"][:, :N * D].float().view(R, H, N // H, D)
    z = torch.einsum("rhgd,rlhd->rhgl", q, k) * D ** -0.5
    if case["cap"]:
        z = case["cap"] * torch.tanh(z / case["cap"])
    seen = torch.arange(most * page, device="cuda") < state["cached"][:, None]
    z = z.masked_fill_(~seen[:, None, None], -math.inf)
    s = state["sink"].float().view(H, N // H, 1) if case["sink"] else torch.tensor(-math.inf, device="cuda")
    top = torch.maximum(z.amax(-1, keepdim=True), s).clamp(min=-1e30)
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True) + torch.exp(s - top)
    p = torch.where(total > 0, p / total, 0.0)
    return {"out": torch.einsum("rhgl,rlhd->rhgd", p, v).flatten(1).to(state["q"].dtype)}


# ---------------------------------------------------------------------------------------------------------- one pass
@torch.no_grad()
def run(state):
    case = state["case"]
    if not own:
        return {"select": _plain_select, "fork": _plain_fork, "tables": _plain_tables, "attend": _plain_attend}[case["kind"]](state)
    from blitz_scale_b200 import ops
    if case["kind"] == "select":
        s = ops.beam_select(state["logits"], state["scores"], beams=case["beams"], n=case["n"], ended=state["ended"])
        return {"score": s.score, "parent": s.parent, "token": s.token, "next_score": s.next_score, "next_parent": s.next_parent,
                "next_token": s.next_token}
    if case["kind"] == "fork":
        page = 2 if case["what"] == "states" else case["page"]
        f = ops.beam_fork(state["table"], state["cached"], state["parents"], state["pool"], page_size=page, num_pages=state["num_pages"])
        ops.copy_pages(state["cache"], f.src, f.dst, f.tokens if case["what"] == "pages" else None, layers=True)
        return {"table": f.table, "cached": f.cached, "src": f.src, "dst": f.dst, "tokens": f.tokens, "cache": state["cache"]}
    if case["kind"] == "tables":
        if case["rows"]:
            t = ops.step_tables(state["table"], state["cached"], state["counts"], page_size=case["page"], tokens=state["tokens"])
            return {"indices": t.indices, "indptr": t.indptr, "last": t.last_page_len, "pos": t.pos, "slot": t.slot, "tok_indptr": t.tok_indptr}
        t = ops.step_tables(state["table"], state["cached"], page_size=case["page"], beams=case["beams"])
        return {"indices": t.indices, "indptr": t.indptr, "last": t.last_page_len, "pos": t.pos, "slot": t.slot, "shared": t.shared}
    return {"out": ops.attn_decode_beams(state["q"], state["kv"], state["indices"], state["indptr"], state["last"], state["shared"],
                                         beams=case["beams"], q_heads=case["q_heads"], kv_heads=case["kv_heads"], head_dim=case["dim"],
                                         page_size=case["page"], softcap=case["cap"], sink=state["sink"], workspace=state["scratch"])}


# ---------------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["kind"] == "select":
        rows, n = case["requests"] * case["beams"], case["requests"] * (case["n"] + case["beams"])
        values = rows * case["vocab"]
        return {"bytes": values * (4 if case["dtype"] == "float32" else 2) + rows * 4 + n * 12, "flops": 4 * values}
    cached, tables, owned, counts, _ = _shape(case)
    H, D, k, R = case["kv_heads"], case["dim"], case["beams"], len(cached)
    width = max(len(t) for t in tables) + 1
    if case["kind"] == "fork":
        page = 2 if case["what"] == "states" else case["page"]
        copied = 0
        for q, parents in enumerate(_parents(case, cached)):
            live = [p for p in parents if p >= 0]
            part = cached[q * k] % page
            copied += (len(live) - len(set(live))) * (part if case["what"] == "pages" else int(part > 0))
        row = 4 * H * D if case["what"] == "pages" else H * page // 16 * 16 * (D + 8 * (D // 32)) if case["what"] == "quantised" else 4 * H * D * D
        pages = sum(len(t) for t in tables)
        # tables of parents and the request's own pages read, tables written
        return {"bytes": 2 * copied * row * case["layers"] + 4 * (pages + sum(b + n - a for a, b, n in owned) + R * width + 6 * R), "flops": R}
    if case["kind"] == "tables":
        pages = sum(-(-(c + n) // case["page"]) for c, n in zip(cached, counts) if c >= 0)
        return {"bytes": 4 * (2 * pages + 5 * R + 2 * sum(counts)), "flops": pages}
    page, seen = case["page"], 0
    for q, n in enumerate(_spread(case, case["prompt"])):
        common = n // page * page
        seen += common + sum(c - common for c in cached[q * k:q * k + k] if c >= 0)
    return {"bytes": seen * 4 * H * D + R * case["q_heads"] * D * 4, "flops": 4 * case["q_heads"] * D * sum(max(c, 0) for c in cached)}


# ---------------------------------------------------------------------------------------------------------- from the definitions
def _exact_select(case, seed):
    state = _select_inputs(case, seed)
    Q, k, V, n = case["requests"], case["beams"], case["vocab"], case["n"]
    ended, found, more = set(state["ended"].tolist()), [], []
    for q in range(Q):
        z = state["logits"][q * k:q * k + k].double()
        v = (torch.log_softmax(z, 1) + state["scores"][q * k:q * k + k].double()[:, None]).flatten()
        v = v.nan_to_num(nan=-math.inf, neginf=-math.inf)
        least = torch.topk(v, min(n, v.numel())).values[-1]
        at = torch.nonzero(v >= least if least > -math.inf else v > -math.inf).flatten()
        got = sorted(zip((-v[at]).tolist(), at.tolist()))[:n]
        got = [(-x, i // V, i % V) for x, i in got]
        found.append(got + [(-math.inf, -1, -1)] * (n - len(got)))
        got = [g for g in got if g[2] not in ended][:k]
        more.append(got + [(-math.inf, -1, -1)] * (k - len(got)))
    out = {}
    for name, rows in (("", found), ("next_", more)):
        for j, what in enumerate(("score", "parent", "token")):
            out[name + what] = torch.tensor([[x[j] for x in r] for r in rows], dtype=torch.float64 if j == 0 else torch.int32)
    return out


def _exact_fork(case, state):
    k, page = case["beams"], 2 if case["what"] == "states" else case["page"]
    old, cached, parents, pool = (state[n].tolist() for n in ("table", "cached", "parents", "pool"))
    W, table, lens, pairs = len(old[0]), [], [], []
    for q, row in enumerate(parents):
        kept, wants, taken, seen = [], [], set(), set()
        for p in row:
            n = cached[q * k + p] if p >= 0 else -1
            mine = old[q * k + p][:n // page] if n >= 0 else []
            fresh = n >= 0 and (n % page == 0 or p in seen)
            if n >= 0 and not fresh:
                mine = mine + [old[q * k + p][n // page]]
            seen.add(p)
            taken.update(mine)
            lens.append(n)
            kept.append(mine)
            wants.append((fresh, old[q * k + p][n // page] if n % page else -1, n % page))
        free = [p for p in pool[q] if p >= 0 and p not in taken]
        for mine, (fresh, page_of, part) in zip(kept, wants):
            at = free.pop(0) if fresh else -1
            pairs.append((page_of, at, part) if fresh and part else (-1, -1, 0))
            mine = mine + [at] if fresh else mine
            table.append(mine + [-1] * (W - len(mine)))
    src, dst, tokens = zip(*pairs)
    cache = state["cache"]
    for a, b, n in pairs:
        if a >= 0 and case["what"] == "pages":
            cache[:, b, :, :n] = cache[:, a, :, :n]
        elif a >= 0:
            cache[:, b] = cache[:, a]
    cache = cache.double() if cache.is_floating_point() else cache
    return {"table": _int32(table), "cached": _int32(lens), "src": _int32(src), "dst": _int32(dst), "tokens": _int32(tokens), "cache": cache}


def _exact_tables(case, state):
    page, k, table, cached = case["page"], case["beams"], state["table"].tolist(), state["cached"].tolist()
    counts = state["counts"].tolist() if case["rows"] else [int(c >= 0) for c in cached]
    indices, indptr, last, pos, slot, tok, lists = [], [0], [], [], [], [0], []
    for row, c, n in zip(table, cached, counts):
        length = c + n if n > 0 else 0
        lists.append(row[:-(-length // page)])
        indices += lists[-1]
        indptr.append(len(indices))
        last.append((length - 1) % page + 1 if length else 0)
        pos += range(c, c + n) if n else [] if case["rows"] else [0]
        slot += [row[i // page] * page + i % page for i in range(c, c + n)] if n else [] if case["rows"] else [-1]
        tok.append(tok[-1] + n)
    indices += [0] * (len(table) * len(table[0]) - len(indices))
    out = {"indices": indices, "indptr": indptr, "last": last, "pos": pos, "slot": slot}
    if case["rows"]:
        out["tok_indptr"] = tok
    else:
        out["shared"] = []
        for q in range(0, len(table), k):
            live = [i for i in range(q, q + k) if counts[i]]
            most = min([(cached[i] + 1) // page for i in live], default=0)
            same = 0
            while same < most and len({lists[i][same] for i in live}) == 1:
                same += 1
            out["shared"].append(same)
    return {n: _int32(x) for n, x in out.items()}


def _exact_attend(case, state):
    H, D, N, page = case["kv_heads"], case["dim"], case["q_heads"], case["page"]
    start, lens, rows = state["indptr"].tolist(), state["cached"].tolist(), []
    for r, n in enumerate(lens):
        if n <= 0:
            rows.append(torch.zeros(N * D, dtype=torch.float64, device="cuda"))
            continue
        kv = state["kv"][state["indices"][start[r]:start[r + 1]].long()].double().transpose(0, 1).reshape(2, -1, H, D)[:, :n]
        z = (state["q"][r, :N * D].double().view(H, N // H, D) @ kv[0].permute(1, 2, 0)) / math.sqrt(D)
        if case["cap"]:
            z = torch.tanh(z / case["cap"]) * case["cap"]
        if case["sink"]:
            z = torch.cat([z, state["sink"].double().view(H, N // H, 1)], 2)
        rows.append((torch.softmax(z, 2)[:, :, :n] @ kv[1].transpose(0, 1)).flatten())
    return {"out": torch.stack(rows)}


@torch.no_grad()
def exact(case, seed):
    if case["kind"] == "select":
        return _exact_select(case, seed)
    return {"fork": _exact_fork, "tables": _exact_tables, "attend": _exact_attend}[case["kind"]](case, prepare(case, seed))
