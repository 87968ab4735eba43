"""Beam search over a paged cache, in plain Python and 64 bits."""
import math

import torch


def select(logits, scores, beams, n, keep, ended=()):
    """[(value, beam, token)] of every request, best first, and those that go on; and all values [requests, beams * vocab]."""
    z = logits.double().cpu()
    v = torch.empty_like(z)
    for r in range(z.shape[0]):
        top = z[r].max()
        v[r] = float(scores[r]) + (z[r] - (top + (z[r] - top).exp().sum().log()))
    v[torch.isnan(v)] = -math.inf
    V = z.shape[1]
    every = v.view(-1, beams * V)
    best, on = [], []
    for row in every:
        order = torch.sort(row, descending=True, stable=True).indices[:n].tolist()
        got = [(row[i].item(), i // V, i % V) for i in order if row[i] > -math.inf]
        best.append(got + [(-math.inf, -1, -1)] * (n - len(got)))
        got = [g for g in got if g[2] not in ended][:keep]
        on.append(got + [(-math.inf, -1, -1)] * (keep - len(got)))
    return best, on, every


def fork(table, cached, parents, pool, page, num_pages):
    """(table, cached, src, dst, tokens) of the children, as lists."""
    Q, k, W = len(parents), len(table) // len(parents), len(table[0])
    out, lens, pairs = [], [], []
    for q in range(Q):
        rows, used, seen = [], set(), set()
        for b in parents[q]:
            n = cached[q * k + b] if 0 <= b < k else -1
            if n < 0 or n // page >= W:
                rows.append(None)
                continue
            old, full = table[q * k + b], n // page
            fresh = n % page == 0 or b in seen
            seen.add(b)
            kept = old[:full] if fresh else old[:full + 1]
            used.update(kept)
            rows.append((n, kept, fresh, old[full] if n % page else -1))
        free = [p for p in pool[q] if 0 <= p < num_pages and p not in used]
        for row in rows:
            if row is None or (row[2] and not free):
                out.append([-1] * W)
                lens.append(-1)
                pairs.append((-1, -1, 0))
                continue
            n, kept, fresh, last = row
            at = free.pop(0) if fresh else -1
            kept = kept + [at] if fresh else kept
            out.append(kept + [-1] * (W - len(kept)))
            lens.append(n)
            pairs.append((last, at, n % page) if fresh and n % page else (-1, -1, 0))
    return [out, lens, *map(list, zip(*pairs))]


def tables(table, cached, counts, page, beams, entries, tokens):
    """The fields of StepTables as lists (counts None: one token for each row)."""
    R, W = len(table), len(table[0])
    indices, indptr, last, pos, slot, tok, took = [], [0], [], [], [], [0], []
    room = True
    for r in range(R):
        n = counts[r] if counts is not None else 1
        if cached[r] < 0 or n <= 0 or cached[r] + n > W * page:
            n = 0
        pages = -(-(cached[r] + n) // page) if n else 0
        room = room and len(indices) + pages <= entries and (counts is None or tok[-1] + n <= tokens)
        if not room:
            n = pages = 0
        took.append(n)
        indices += table[r][:pages]
        indptr.append(len(indices))
        last.append((cached[r] + n - 1) % page + 1 if n else 0)
        tok.append(tok[-1] + n)
        at = list(range(cached[r], cached[r] + n)) if n else [] if counts is not None else [None]
        pos += [0 if i is None else i for i in at]
        slot += [-1 if i is None or table[r][i // page] < 0 else table[r][i // page] * page + i % page for i in at]
    indices += [0] * (entries - len(indices))
    if counts is not None:
        pos += [0] * (tokens - len(pos))
        slot += [-1] * (tokens - len(slot))
    shared = None
    if beams:
        shared = []
        for q in range(0, R, beams):
            live = [r for r in range(q, q + beams) if took[r]]
            most, same = min([(cached[r] + took[r]) // page for r in live], default=0), 0
            while same < most and len({table[r][same] for r in live}) == 1:
                same += 1
            shared.append(same)
    return [indices, indptr, last, pos, slot, tok if counts is not None else None, shared]


def attend(q, kv, lists, lengths, q_heads, kv_heads, dim, scale=None, cap=0.0, sink=None):
    """[rows, q_heads * dim] in 64 bits; lists: pages of every row."""
    rows = []
    for r, (pages, n) in enumerate(zip(lists, lengths)):
        if n == 0:
            rows.append(torch.zeros(q_heads * dim, dtype=torch.float64))
            continue
        x = kv[torch.tensor(pages, device=kv.device)].double().cpu().transpose(0, 1).reshape(2, -1, kv_heads, dim)[:, :n]
        z = q[r, :q_heads * dim].double().cpu().view(kv_heads, -1, dim) @ x[0].permute(1, 2, 0) * (dim ** -0.5 if scale is None else scale)
        if cap:
            z = cap * torch.tanh(z / cap)
        if sink is not None:
            z = torch.cat([z, sink.double().cpu().view(kv_heads, -1, 1)], 2)
        rows.append((torch.softmax(z, 2)[:, :, :n] @ x[1].transpose(0, 1)).flatten())
    return torch.stack(rows)
