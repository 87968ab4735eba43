"""A key/value cache held in 4 bits, and the attention that reads it: one pass of an operator on one GPU.

Kinds of a case: `store` (rows of keys and values are quantised into the paged cache, and read back), `pages` (whole pages are read
back in the layout of a 16-bit cache, as a prompt's later portions or a migration need them), `decode` (attention of one token of
every sequence) and `portion` (causal attention of portions of prompts, which the cache holds already, with whatever came before).

The cache of a layer is a tensor of bytes [pages, kv_heads, page / 16, block].  A block is 16 tokens of one head: codes of the keys,
their scales, codes of the values, their scales.  A group of `group` dimensions of a head has an offset z and a scale s in bf16, and a
dimension x is z + s c with a code c of 4 bits:

    z = min x, rounded down to bf16;  s = (max x - z) / 15, rounded up;  c = rint((x - z) / s), ties to even, in 0 .. 15 (s = 0: 0)

Keys: token after token, dim / 2 bytes each; dimension 32 w + 8 l + i is in nibble i of 32-bit word l dim/32 + w.  Values: dimension
64 h + 16 m + 8 n + g of token 4 a + 2 x + y is nibble n (0: the low one) of byte h 512 + g 64 + a 16 + 4 m + 2 y + x (heads of 64: h = 0).
Scales: per token the groups' s, then their z.

Prepared caches hold quantised numbers of the sizes that keys and values have in models: a few dimensions of the keys are several
times larger than the others, and scores are of order one.
"""
import math
import random

import torch

own = False
PAGE = 64
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


# ---------------------------------------------------------------------------------------------------------- cases
def _case(name, kind, sequences, tokens, *, rows=0, heads=(32, 8), dim=128, group=32, page=PAGE, ragged=False, window=0, keep=0, cap=0.0,
          sink=False, dtype="bfloat16"):
    """`tokens`: of the caches of all sequences (store and pages: rows); `rows`: of the portions, each the end of its sequence."""
    return {"name": name, "kind": kind, "sequences": sequences, "tokens": tokens, "rows": rows, "q_heads": heads[0], "kv_heads": heads[1],
            "dim": dim, "group": group, "page": page, "ragged": ragged, "window": window, "keep": keep, "cap": cap, "sink": sink,
            "dtype": dtype}


def listed():
    return [
        # one user's request: the key and value of a token
        _case("store 1", "store", 1, 1),
        # a decode batch: each token in a page of its own
        _case("store 256", "store", 256, 256, group=64),
        # a full pass of prompts, small pages, the second 16-bit type
        _case("store 8192", "store", 9, 8192, ragged=True, page=16, dtype="float16"),
        # a short prefix read back for the portion behind it
        _case("pages 37", "pages", 1, 37 * 64, heads=(16, 4), dim=64, group=64),
        # the caches of a batch that moves to a replica with a 16-bit cache
        _case("pages 1024", "pages", 1, 1024 * 64),
        # one user's request, token by token: latency
        _case("decode 1", "decode", 1, 977),
        # one long context
        _case("decode 1 long", "decode", 1, 100003, group=128),
        # the headline benchmark's batch
        _case("decode 256", "decode", 256, 256 * 512),
        # what continuous batching makes of traffic: requests of very different ages
        _case("decode 61 ragged", "decode", 61, 61 * 1100, ragged=True, group=64, dtype="float16"),
        # windowed attention with kept tokens, a soft cap and a sink, small heads and pages
        _case("decode 24 window", "decode", 24, 24 * 1500, ragged=True, heads=(16, 4), dim=64, page=16, window=1024, keep=4, cap=50.0, sink=True),
        # chunked prefill: a portion of a long prompt behind what is cached of it
        _case("portion 1531", "portion", 1, 1531 + 2311, rows=1531),
        # a full prefill batch of prompts of unequal lengths
        _case("portion 8192 ragged", "portion", 9, 8192, rows=8192, ragged=True, group=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "store", "pages", "decode", "decode", "decode", "portion", "portion"])
    dim = rng.choice([128, 128, 64])
    kv = rng.choice([1, 2, 4, 8, 8])
    more = dict(heads=(kv * rng.choice([1, 2, 4, 4, 5, 8]), kv), dim=dim, group=rng.choice([g for g in (32, 64, 128) if g <= dim]),
                page=rng.choice([16, 64, 64, 128]), ragged=rng.random() < 0.7, dtype=rng.choice(["bfloat16", "bfloat16", "float16"]))
    if kind == "store":
        tokens = _log(rng, 1, 8192)
        case = _case("", kind, min(tokens, _log(rng, 1, 256)), tokens, **more)
    elif kind == "pages":
        case = _case("", kind, 1, more["page"] * max(1, _log(rng, 1, 65536) // more["page"]), **more)
    else:
        if rng.random() < 0.3:
            more.update(window=_log(rng, 64, 4096), keep=rng.choice([0, 4, 37]))
        if rng.random() < 0.3:
            more.update(cap=50.0)
        if rng.random() < 0.3:
            more.update(sink=True)
        if kind == "decode":
            n = _log(rng, 1, 256)
            case = _case("", kind, n, n * _log(rng, 1, min(60000, 131072 // n)), **more)
        else:
            n = rng.choice([1, 1, 2, 4, 8])
            rows = max(n, _log(rng, 24, 4096))
            case = _case("", kind, n, rows + rng.choice([0, _log(rng, 16, 4096)]), rows=rows, **more)
    del case["name"]
    return case


def _spread(case, total):
    """`total` over the sequences, one at least for each: equal, or spread over a factor of sixteen.  A matter of the case alone."""
    n = case["sequences"]
    rng = random.Random(n * 1000003 + total)
    w = [math.exp(rng.uniform(0.0, math.log(16.0))) if case["ragged"] else 1.0 for _ in range(n)]
    out = [max(1, int(total * x / sum(w))) for x in w]
    while sum(out) != total:
        i = rng.randrange(n)
        out[i] += 1 if sum(out) < total else -1 if out[i] > 1 else 0
    return out


def _lengths(case):
    """(tokens of every sequence in the cache, rows of it in the pass)"""
    if case["kind"] == "decode":
        kv = _spread(case, case["tokens"])
        return kv, [1] * len(kv)
    if case["kind"] == "portion":
        rows, before = _spread(case, case["rows"]), case["tokens"] - case["rows"]
        more = [before // len(rows) + (i < before % len(rows)) for i in range(len(rows))]
        return [a + b for a, b in zip(rows, more)], rows
    rows = _spread(case, case["tokens"])
    return rows, rows


# ---------------------------------------------------------------------------------------------------------- the cache's bytes
def _bf16_down(x):
    y = x.to(torch.bfloat16)
    return torch.where(y.float() > x, torch.nextafter(y, torch.full_like(y, -math.inf)), y)


def _bf16_up(x):
    return -_bf16_down(-x)


def _quantise(x, group):
    """x [..., dim] in 16 bits -> codes [..., dim], scales and offsets [..., groups] (fp32 with bf16 values)."""
    x = x.float().unflatten(-1, (-1, group))
    z = _bf16_down(x.amin(-1)).float()
    s = _bf16_up((x.amax(-1) - z) / torch.full_like(z, 15.0)).float()       # (by a number, a GPU would take its reciprocal)
    c = torch.round((x - z[..., None]) / torch.where(s > 0, s, 1.0)[..., None]).clamp(0, 15)
    return torch.where(s[..., None] > 0, c, 0.0).flatten(-2), s, z


def _values(c, s, z, group):
    return (c.unflatten(-1, (-1, group)) * s[..., None] + z[..., None]).flatten(-2)


def _words(s, z):
    """Scales and offsets [blocks, 16, groups] as bytes."""
    return torch.cat([s, z], -1).to(torch.bfloat16).flatten(1).contiguous().view(torch.uint8)


def _blocks(k, v, group):
    """Blocks [n, bytes] of keys and values [n, 16, dim]."""
    n, _, dim = k.shape
    (kc, ks, kz), (vc, vs, vz) = _quantise(k, group), _quantise(v, group)
    kc, vc = kc.to(torch.uint8), vc.to(torch.uint8)
    kc = kc.view(n, 16, dim // 32, 4, 4, 2).transpose(2, 3)                      # token, lane, word, byte, nibble
    vc = vc.view(n, 4, 2, 2, dim // 64, 4, 2, 8).permute(0, 4, 7, 1, 5, 3, 2, 6)  # half, row, quad, tile, y, x, nibble
    join = lambda c: (c[..., 0] + 16 * c[..., 1]).reshape(n, -1)  # noqa: E731
    return torch.cat([join(kc), _words(ks, kz), join(vc), _words(vs, vz)], 1)


def _read(blocks, dim, group):
    """Keys and values [n, 16, dim] (fp32) of blocks [n, bytes]."""
    n, codes = blocks.shape[0], 8 * dim
    part = codes + 64 * (dim // group)
    nibbles = lambda b: torch.stack([b & 15, b >> 4], -1).float()  # noqa: E731
    kc = nibbles(blocks[:, :codes]).view(n, 16, 4, dim // 32, 4, 2).transpose(2, 3).reshape(n, 16, dim)
    vc = nibbles(blocks[:, part:part + codes]).view(n, dim // 64, 8, 4, 4, 2, 2, 2).permute(0, 3, 6, 5, 1, 4, 7, 2).reshape(n, 16, dim)
    words = lambda at: blocks[:, at + codes:at + part].contiguous().view(torch.bfloat16).float().view(n, 16, 2, dim // group)  # noqa: E731
    kw, vw = words(0), words(part)
    return _values(kc, kw[:, :, 0], kw[:, :, 1], group), _values(vc, vw[:, :, 0], vw[:, :, 1], group)


# ---------------------------------------------------------------------------------------------------------- inputs
def _rows(gen, n, case, what):
    """Rows of queries, keys or values as models have them."""
    H, D = case["q_heads" if what == "q" else "kv_heads"], case["dim"]
    x = torch.randn(n, H, D, generator=gen, device="cuda")
    if what == "k":
        x[:, :, ::37] *= 4.0        # (dimensions that stick out)
        x += 0.5 * torch.randn(1, H, D, generator=gen, device="cuda")
    return x.to(DTYPES[case["dtype"]])


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    H, D, page, group, dt = case["kv_heads"], case["dim"], case["page"], case["group"], DTYPES[case["dtype"]]
    kv, rows = _lengths(case)
    held = [-(-n // page) for n in kv]
    P = sum(held)
    place = torch.randperm(P + 3, generator=torch.Generator().manual_seed(seed))[:P].to(torch.int32).cuda()    # pages, as a pool hands them out
    state = {"case": case, "pages": place}
    block = 16 * (D + 8 * (D // group))
    pool = torch.zeros(P + 3, H, page // 16, block, dtype=torch.uint8, device="cuda")
    state["pool"] = pool
    n = torch.tensor(kv)
    first = torch.cat([torch.zeros(1, dtype=torch.long), torch.tensor(held).cumsum(0)])
    seq = torch.repeat_interleave(torch.arange(len(kv)), n)
    pos = torch.arange(int(n.sum())) - torch.repeat_interleave(n.cumsum(0) - n, n)
    if case["kind"] == "store":
        slot = place.cpu()[first[seq] + pos // page].long() * page + pos % page
        state["slot"] = slot.to(torch.int32).cuda()
        # the keys and values of a projection's rows [queries | keys | values]
        T = slot.numel()
        qkv = torch.cat([torch.zeros(T, case["q_heads"] * D, dtype=dt, device="cuda"), _rows(gen, T, case, "k").flatten(1), _rows(gen, T, case, "v").flatten(1)], 1)
        state.update(k=qkv[:, case["q_heads"] * D:][:, :H * D], v=qkv[:, -H * D:])
        return state
    for a in range(0, P, 1024):
        at = place[a:a + 1024].long()
        k, v = (_rows(gen, at.numel() * page, case, w).view(-1, page // 16, 16, H, D).permute(0, 3, 1, 2, 4).reshape(-1, 16, D) for w in "kv")
        pool[at] = _blocks(k, v, group).view(at.numel(), H, page // 16, block)
    if case["kind"] == "pages":
        return state
    T = sum(rows)
    q = torch.zeros(T, (case["q_heads"] + 2 * H) * D, dtype=dt, device="cuda")
    q[:, :case["q_heads"] * D] = _rows(gen, T, case, "q").flatten(1)
    state.update(q=q, kv=kv, rows=rows, indptr=first.to(torch.int32).cuda(),
                 last=torch.tensor([(m - 1) % page + 1 for m in kv], dtype=torch.int32, device="cuda"),
                 kv_dev=n.cuda(), rows_dev=torch.tensor(rows).cuda(),
                 sink=torch.randn(case["q_heads"], generator=gen, device="cuda").to(dt) if case["sink"] else None)
    if own:
        # what a serving process keeps: the records of a pass's tiles, scratch
        from blitz_scale_b200 import ops
        if case["kind"] == "portion":
            state["work"] = ops.prefill_work_list(rows, kv, page, "cuda")
        else:
            state["scratch"] = torch.zeros(ops.quant_attn_workspace_bytes(len(kv), case["q_heads"], D, "cuda"), dtype=torch.uint8, device="cuda")
    return state


# ---------------------------------------------------------------------------------------------------------- plain forms
def _padded(state):
    """Keys and values [sequences, longest, heads, dim] (fp32) of the sequences' pages; behind a sequence's end those of some page."""
    case = state["case"]
    H, D, page = case["kv_heads"], case["dim"], case["page"]
    most = -(-max(state["kv"]) // page)
    at = (state["indptr"][:-1, None] + torch.arange(most, device="cuda")).clamp(max=state["pages"].numel() - 1)
    b = state["pool"][state["pages"][at.long()].long()]                        # [sequences, pages, heads, blocks, bytes]
    x = _read(b.flatten(0, 3), D, case["group"])
    return (t.view(*b.shape[:4], 16, D).permute(0, 1, 3, 4, 2, 5).reshape(b.shape[0], most * page, H, D) for t in x)


def _attention(state):
    case = state["case"]
    H, D, Q = case["kv_heads"], case["dim"], case["q_heads"]
    k, v = _padded(state)
    n, longest = state["rows_dev"], max(state["rows"])
    i = torch.arange(longest, device="cuda")
    row = (n.cumsum(0) - n)[:, None] + i                                       # rows of each sequence, padded
    real = i < n[:, None]
    q = state["q"][row.clamp(max=state["q"].shape[0] - 1), :Q * D].float().view(len(n), longest, H, Q // H, D)
    z = torch.einsum("slhgd,skhd->shglk", q, k) * D ** -0.5
    if case["cap"]:
        z = case["cap"] * torch.tanh(z / case["cap"])
    j, at = torch.arange(k.shape[1], device="cuda"), (state["kv_dev"] - n)[:, None] + i
    seen = j <= at[:, :, None]
    if case["window"]:
        seen &= (j > at[:, :, None] - case["window"]) | (j < case["keep"])
    z = z.masked_fill_(~seen[:, None, None], -math.inf)
    if case["sink"]:
        s = state["sink"].float().view(1, H, Q // H, 1, 1)
        top = torch.maximum(z.amax(-1, keepdim=True), s)
        p = torch.exp(z - top)
        p = p / (p.sum(-1, keepdim=True) + torch.exp(s - top))
    else:
        p = torch.exp(z - z.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
    o = torch.einsum("shglk,skhd->slhgd", p, v).flatten(2)
    return o[real].to(state["q"].dtype)


def _plain(state):
    case = state["case"]
    H, D, page = case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "store":
        dt = state["k"].dtype
        k, v = (_values(*_quantise(x.unflatten(1, (H, D)), case["group"]), case["group"]).to(dt) for x in (state["k"], state["v"]))
        return {"k": k, "v": v}
    if case["kind"] == "pages":
        b = state["pool"][state["pages"].long()]
        k, v = _read(b.flatten(0, 2), D, case["group"])
        both = torch.stack([x.view(*b.shape[:3], 16, D).permute(0, 2, 3, 1, 4).reshape(-1, page, H, D) for x in (k, v)], 1)
        return {"cache": both.to(DTYPES[case["dtype"]])}
    return {"out": _attention(state)}


# ---------------------------------------------------------------------------------------------------------- one pass
@torch.no_grad()
def run(state):
    if not own:
        return _plain(state)
    from blitz_scale_b200 import ops
    case = state["case"]
    cache = ops.QuantKV(state["pool"], case["dim"], case["group"])
    if case["kind"] == "store":
        ops.quant_kv_store(state["k"], state["v"], state["slot"], cache)
        k, v = ops.quant_kv_load(cache, state["slot"], dtype=state["k"].dtype)
        return {"k": k, "v": v}
    if case["kind"] == "pages":
        return {"cache": ops.quant_kv_pages(cache, state["pages"], dtype=DTYPES[case["dtype"]])}
    more = dict(q_heads=case["q_heads"], kv_heads=case["kv_heads"], head_dim=case["dim"], page_size=case["page"], window=case["window"],
                keep_first=case["keep"], softcap=case["cap"], sink=state["sink"])
    if case["kind"] == "decode":
        return {"out": ops.attn_decode(state["q"], cache, state["pages"], state["indptr"], state["last"], num_splits=0, workspace=state["scratch"], **more)}
    return {"out": ops.attn_prefill_paged(state["q"], cache, state["pages"], state["work"], **more)}


# ---------------------------------------------------------------------------------------------------------- what a pass cannot do without
def _seen(case, length, rows):
    """(keys that the last `rows` positions of a sequence see, counted for each; how many different ones)"""
    w, keep = case["window"], case["keep"]
    first = length - rows
    if not w:
        return rows * first + rows * (rows + 1) // 2, length
    pairs = sum(min(i + 1, w) + min(keep, max(0, i + 1 - w)) for i in range(first, length))
    low = max(0, first + 1 - w)
    return pairs, length - low + min(keep, low)


def work(case):
    H, D, Q = case["kv_heads"], case["dim"], case["q_heads"]
    token = 2 * H * (D // 2 + 4 * (D // case["group"]))       # bytes of a token's keys and values in 4 bits
    if case["kind"] == "store":
        return {"bytes": case["tokens"] * (2 * 4 * H * D + token), "flops": case["tokens"] * H * D * 2 * 6}
    if case["kind"] == "pages":
        return {"bytes": case["tokens"] * (4 * H * D + token), "flops": case["tokens"] * H * D * 2 * 2}
    kv, rows = _lengths(case)
    seen = [_seen(case, a, b) for a, b in zip(kv, rows)]
    return {"bytes": sum(s[1] for s in seen) * token + sum(rows) * Q * D * 4, "flops": 4 * Q * D * sum(s[0] for s in seen)}


# ---------------------------------------------------------------------------------------------------------- in 64 bits
def _exact_rows(x, case):
    """Keys or values [rows, heads x dim] as the cache holds them, from the definition in 64 bits."""
    x = x.double().view(x.shape[0], case["kv_heads"], -1, case["group"])

    def below(a):       # the largest number of 8 significant bits that is not above a
        m, e = torch.frexp(a)
        return torch.ldexp(torch.floor(m * 256), e - 8)
    z = below(x.min(-1, keepdim=True).values)
    s = -below((z - x.max(-1, keepdim=True).values) / torch.full_like(z, 15.0))
    return (z + s * torch.round((x - z) / s.clamp(min=1e-300)).clamp(0, 15)).flatten(1)


def _exact_cache(state, tokens):
    """Keys and values [tokens, heads, dim] in 64 bits at places `tokens` (page, offset): every code by its address."""
    case = state["case"]
    H, D, group = case["kv_heads"], case["dim"], case["group"]
    G, codes = D // group, 8 * D
    bytes_ = state["pool"].reshape(-1)
    page, off = (t.cuda() for t in tokens)
    base = (page[:, None] * H + torch.arange(H, device="cuda")) * (case["page"] // 16) + (off // 16)[:, None]
    base = (base * state["pool"].shape[-1])[:, :, None]
    t, d = (off % 16)[:, None, None], torch.arange(D, device="cuda")
    word = (d // 8 % 4) * (D // 32) + d // 32
    k_at, k_nib = t * (D // 2) + word * 4 + d % 8 // 2, d % 2
    v_at, v_nib = (d // 64) * 512 + (d % 8) * 64 + (t // 4) * 16 + (d // 16 % 4) * 4 + t % 2 * 2 + t // 2 % 2, d // 8 % 2

    def number(at):     # bf16 at a byte address
        return ((bytes_[at].int() | bytes_[at + 1].int() << 8) << 16).view(torch.float32).double()
    out = []
    for start, at, nib in ((0, k_at, k_nib), (codes + 64 * G, v_at, v_nib)):
        c = (bytes_[base + start + at].int() >> (4 * nib)) & 15
        s_at = base + start + codes + t * 4 * G + 2 * (d // group)
        out.append(number(s_at + 2 * G) + number(s_at) * c.double())
    return out


@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    H, D, Q, page = case["kv_heads"], case["dim"], case["q_heads"], case["page"]
    if case["kind"] == "store":
        return {n: _exact_rows(state[n], case).view(-1, H, D) for n in "kv"}
    if case["kind"] == "pages":
        n = state["pages"].numel()
        k, v = _exact_cache(state, (state["pages"].long().repeat_interleave(page), torch.arange(page).repeat(n)))
        return {"cache": torch.stack([k.view(n, page, H, D), v.view(n, page, H, D)], 1)}
    out = []
    ends = torch.tensor(state["rows"]).cumsum(0).tolist()
    starts = state["indptr"].tolist()
    for s, (length, rows) in enumerate(zip(state["kv"], state["rows"])):
        j = torch.arange(length)
        k, v = _exact_cache(state, (state["pages"].long().cpu()[starts[s] + j // page], j % page))
        q = state["q"][ends[s] - rows:ends[s], :Q * D].double().view(rows, Q, D)
        i = torch.arange(length - rows, length)[:, None]
        hidden = j > i
        if case["window"]:
            hidden |= (j <= i - case["window"]) & (j >= case["keep"])
        o = torch.empty(rows, Q, D, dtype=torch.float64, device="cuda")
        for h in range(Q):
            z = q[:, h] @ k[:, h // (Q // H)].t() / math.sqrt(D)
            if case["cap"]:
                z = torch.tanh(z / case["cap"]) * case["cap"]
            z[hidden.cuda()] = -math.inf
            if case["sink"]:
                z = torch.cat([z, state["sink"][h].double().expand(rows, 1)], 1)
            o[:, h] = torch.softmax(z, 1)[:, :length] @ v[:, h // (Q // H)]
        out.append(o.flatten(1))
    return {"out": torch.cat(out)}
