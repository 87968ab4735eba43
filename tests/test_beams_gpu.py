"""Beam search over a paged cache: selection, tables, copies and attention against plain forms in 64 bits."""
import math
import random

import pytest
import torch

import beams_plain as plain
from blitz_scale_b200 import ops

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

# Exponentials to 2^-22 and arguments within 20 of the largest to 20 x 2^-23 (what is further away weighs e^-20 at most); about 30 additions in fp32: the log of
# their sum is off by 5e-6 at most, a score by that and its rounding.
LSE = 5e-6


def _same_selection(got, want, on, every, V):
    """Candidates in the order of their values; another order only where values of different beams are within what the sums may be off by."""
    for (score, parent, token), rows in (((got.score, got.parent, got.token), want), ((got.next_score, got.next_parent, got.next_token), on)):
        score, parent, token = score.cpu().tolist(), parent.cpu().tolist(), token.cpu().tolist()
        for q, row in enumerate(rows):
            for i, (v, b, t) in enumerate(row):
                if v == -math.inf:
                    assert (score[q][i], parent[q][i], token[q][i]) == (-math.inf, -1, -1)
                    continue
                assert abs(score[q][i] - v) <= LSE + 2.0 ** -24 * abs(v), (q, i, score[q][i], v)
                if (parent[q][i], token[q][i]) != (b, t):
                    assert parent[q][i] != b and abs(every[q][parent[q][i] * V + token[q][i]].item() - v) <= 2 * LSE, (q, i)


def _select(logits, scores, beams, n=0, keep=0, ended=None):
    got = ops.beam_select(logits, scores, beams, n=n, keep=keep, ended=ended)
    ops.check_status()
    n = n or 2 * beams
    want, on, every = plain.select(logits, scores, beams, n, keep or min(beams, n), set() if ended is None else set(ended.tolist()))
    _same_selection(got, want, on, every, logits.shape[1])
    return got


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("V,beams,n", [(1, 1, 1), (1, 3, 5), (5, 2, 12), (7, 1, 2), (127, 4, 8), (1003, 5, 10), (16384, 2, 16), (16389, 3, 17), (50257, 8, 33), (131072, 4, 64), (152064, 1, 2)])
def test_select_sizes(dtype, V, beams, n):
    g = torch.Generator("cuda").manual_seed(V + n)
    rows = 3 * beams
    z = (3.0 * torch.randn(rows, V, generator=g, device="cuda")).to(dtype)
    s = -30.0 * torch.rand(rows, generator=g, device="cuda")
    _select(z, s, beams, n, ended=torch.randint(0, V, (3,), generator=g, device="cuda").to(torch.int32))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("offset,pitch", [(1, 1005), (3, 1009), (0, 1003), (5, 1024), (8, 4099)])
def test_select_rows_anywhere(dtype, offset, pitch):
    """Rows that begin and end off the 16-byte boundaries, between numbers that would win."""
    room = torch.full((offset + 6 * pitch + 16,), 1000.0, dtype=dtype, device="cuda")
    z = room[offset:offset + 6 * pitch].view(6, pitch)[:, :1003]
    z.copy_(torch.randn(6, 1003, generator=torch.Generator("cuda").manual_seed(pitch), device="cuda"))
    _select(z, torch.zeros(6, device="cuda"), 3)


@pytest.mark.parametrize("what", ["equal", "few values", "rising", "falling", "zeros of both signs", "one group", "minus infinity", "lowest", "one row lowest", "huge"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_select_values(dtype, what):
    """Ties (the lowest token), many candidates of one group of threads, masks of minus infinity or the type's lowest number."""
    V, beams, n = 40001, 2, 16
    g = torch.Generator("cuda").manual_seed(3)
    z = torch.randn(4, V, generator=g, device="cuda")
    if what == "equal":
        z.fill_(1.5)
    elif what == "few values":
        z = torch.round(z * 2)
    elif what == "rising":
        z = (torch.arange(V, device="cuda") / 64).floor().expand(4, -1).clone() / 32
    elif what == "falling":
        z = -(torch.arange(V, device="cuda") / 64).floor().expand(4, -1).clone() / 32
    elif what == "zeros of both signs":
        z = torch.where(z > 0, 0.0, -0.0)
    elif what == "one group":
        at = torch.arange(V, device="cuda") // 8 % 256 < 64
        z = torch.where(at, torch.round(z) + 20, z)
    elif what == "minus infinity":
        z[:, torch.rand(V, generator=g, device="cuda") < 0.9999] = -math.inf
    elif what == "lowest":
        z[:, torch.rand(V, generator=g, device="cuda") < 0.999] = torch.finfo(dtype).min
    elif what == "one row lowest":
        z[1] = torch.finfo(dtype).min
        z[2] = -math.inf
    else:
        z = z * 1e37
    got = _select(z.to(dtype), torch.tensor([-1.0, -1.0, -2.0, -0.5], device="cuda"), beams, n)
    if what == "equal":
        assert got.token[0].tolist() == list(range(16)) and got.parent[0].tolist() == [0] * 16


def test_select_no_numbers():
    """A row with a NaN or +inf has no candidates; the others of its request keep theirs."""
    z = torch.randn(8, 20000, generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    z[0, 17], z[3, 19999], z[4], z[5] = math.nan, math.inf, -math.inf, math.nan
    got = _select(z, torch.tensor([-1.0, -2.0, -3.0, -4.0, -1.0, -2.0, -math.inf, math.nan], device="cuda"), 2, 8)
    assert got.parent.tolist() == [[1] * 8, [0] * 8, [-1] * 8, [-1] * 8]
    for dtype in (BF, HF):
        _select(z.to(dtype), torch.zeros(8, device="cuda"), 4, 8)


def test_select_rows_of_one_memory():
    """Rows that are one row, as at the beginning of a search, and rows of a narrower view."""
    z = torch.randn(1, 3001, generator=torch.Generator("cuda").manual_seed(2), device="cuda").to(BF)
    got = _select(z.expand(4, -1), torch.tensor([0.0, -1.0, -math.inf, -0.5], device="cuda"), 4)
    assert got.token[0, 0] == z[0].argmax() and got.parent[0, 0] == 0
    _select(z.view(3001)[:3000].view(4, 750)[:, 3:], torch.zeros(4, device="cuda"), 2, 9, 4)


def test_select_ended_tokens():
    z = torch.full((4, 300), -5.0, device="cuda")
    z[:, 7], z[:, 9], z[:, 11] = 5.0, 4.0, 3.0
    z[2:] = -math.inf
    z[2, 7], z[3, 7], z[3, 9] = 1.0, 2.0, 1.0
    got = _select(z, torch.tensor([0.0, -1.0, 0.0, 0.0], device="cuda"), 2, 6, 3, ended=i32([7, 8]))
    assert got.next_token.tolist() == [[9, 11, 9], [9, -1, -1]] and got.next_parent.tolist() == [[0, 0, 1], [1, -1, -1]]
    got = _select(z, torch.zeros(4, device="cuda"), 2, ended=torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert got.next_token.tolist() == [[7, 7], [7, 7]]


def test_select_captured_on_another_stream_and_twice():
    z, s = torch.randn(40, 30011, device="cuda").to(BF), -torch.rand(40, device="cuda")
    want = ops.beam_select(z, s, 5)
    out = ops.BeamStep(*(torch.empty_like(t) for t in want))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            ops.beam_select(z, s, 5, out=out)
        for _ in range(3):
            for t in out:
                t.fill_(7)
            graph.replay()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, out))
    z.copy_(z.flip(0))
    s.copy_(s.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ops.beam_select(z, s, 5), out))
    empty = ops.beam_select(z[:0], s[:0], 5)
    assert empty.score.shape == (0, 10) and empty.next_token.shape == (0, 5)


# ---------------------------------------------------------------------------------------------------------- tables of the beams that go on
def _fork_case(rng, Q, k, to, page, W, dead=0.2):
    """Tables as a search makes them: pages at the beginning shared, later ones of a row's own."""
    pool, table, cached, num = [], [], [], 0
    for _ in range(Q):
        n = rng.randrange(0, W * page)
        common = rng.randrange(0, n // page + 1)
        shared = list(range(num, num + common))
        num += common
        mine = []
        for _ in range(k):
            own = list(range(num, num + -(-n // page) - common))
            num += len(own)
            mine += own
            live = rng.random() >= dead
            table.append((shared + own + [-1] * W)[:W] if live else [-1] * W)
            cached.append(n if live else -1)
        spare = list(range(num, num + to))
        num += to
        pool.append(shared + mine + spare)
    most = max(len(p) for p in pool) + 2
    perm = list(range(num))
    rng.shuffle(perm)
    name = lambda p: perm[p] if p >= 0 else p  # noqa: E731
    for p in pool:
        rng.shuffle(p)
    pool = [[name(x) for x in p] + [-1] * (most - len(p)) for p in pool]
    table = [[name(x) for x in t] for t in table]
    parents = [[rng.choice([-1] + list(range(k)) * 3) for _ in range(to)] for _ in range(Q)]
    return table, cached, parents, pool, num


@pytest.mark.parametrize("Q,k,to,page,W", [(1, 1, 1, 16, 1), (3, 4, 4, 16, 3), (5, 8, 8, 64, 40), (2, 1, 6, 16, 5), (7, 5, 2, 128, 9), (1, 64, 64, 16, 7), (40, 4, 4, 2, 1), (2, 3, 3, 64, 1700),
                                           (3, 2, 2, 48, 11), (6, 4, 4, 1, 20)])
def test_fork(Q, k, to, page, W):
    for seed in range(4):
        case = _fork_case(random.Random(seed * 100 + W), Q, k, to, page, W, dead=0.2 * (seed % 2))
        table, cached, parents, pool, num = case
        got = ops.beam_fork(i32(table), i32(cached), i32(parents), i32(pool), page_size=page, num_pages=num)
        ops.check_status()
        want = plain.fork(table, cached, parents, pool, page, num)
        for g, w, name in zip(got, want, ops.BeamFork._fields):
            assert g.tolist() == w, name
        # a table and a pool that are part of wider ones
        wide = torch.full((Q * k, W + 3), 7, dtype=torch.int32, device="cuda")
        wide[:, 1:W + 1] = i32(table)
        more = torch.full((Q, len(pool[0]) + 5), 3, dtype=torch.int32, device="cuda")
        more[:, 2:2 + len(pool[0])] = i32(pool)
        out = ops.BeamFork(*(torch.full_like(t, 99) for t in got))
        ops.beam_fork(wide[:, 1:W + 1], i32(cached), i32(parents), more[:, 2:2 + len(pool[0])], page_size=page, num_pages=num, out=out)
        assert all(torch.equal(a, b) for a, b in zip(got, out))


def test_fork_without_pages_or_room():
    # two children of a parent with a partly filled page, and no page for the second
    table, more = i32([[3, 1], [2, -1]]), dict(page_size=16, num_pages=8)
    got = ops.beam_fork(table, i32([20, 9]), i32([[0, 0]]), i32([[3, 1]]), **more)
    with pytest.raises(RuntimeError, match="no page left"):
        ops.check_status()
    assert got.table.tolist() == [[3, 1], [-1, -1]] and got.cached.tolist() == [20, -1] and got.src.tolist() == [-1, -1] and got.dst.tolist() == [-1, -1]
    # a full table, a parent that there is not, a page that there is not
    got = ops.beam_fork(table, i32([32, 9]), i32([[0, 1]]), i32([[5, 6]]), **more)
    with pytest.raises(RuntimeError, match="size beyond"):
        ops.check_status()
    assert got.table.tolist() == [[-1, -1], [2, -1]] and got.cached.tolist() == [-1, 9]
    got = ops.beam_fork(table, i32([20, 9]), i32([[2, 1]]), i32([[5, 6]]), **more)
    with pytest.raises(RuntimeError, match="index"):
        ops.check_status()
    assert got.cached.tolist() == [-1, 9]
    ops.beam_fork(i32([[100, 1]]), i32([20]), i32([[0]]), i32([[1000000, 6]]), **more)
    with pytest.raises(RuntimeError, match="index"):
        ops.check_status()
    with pytest.raises(ValueError, match="shares memory"):
        ops.beam_fork(table, i32([20, 9]), i32([[0, 1]]), i32([[5, 6]]), **more, out=ops.BeamFork(table, *i32([[0] * 2] * 4).unbind()))


# ---------------------------------------------------------------------------------------------------------- copies
PAIRS = [(3, 9, 5), (-1, 4, 5), (2, -1, 16), (0, 11, 16), (7, 1, 1), (8, 6, 0), (5, 5, 3), (10, 12, 99)]


@pytest.mark.parametrize("shape,dtype,layers,by_token", [
    ((3, 14, 2, 16, 2, 64), BF, True, True), ((14, 2, 16, 3, 20), HF, False, True), ((14, 2, 16, 1, 13), HF, False, True), ((2, 14, 2, 16, 8, 128), BF, True, False),
    ((14, 7, 3), torch.uint8, False, False), ((14, 33, 70), F32, False, False), ((4, 14, 3, 128, 96), F32, True, False), ((2, 14, 1, 1, 400), torch.uint8, True, False), ((14,), F32, False, False)])
def test_copies(shape, dtype, layers, by_token):
    g = torch.Generator("cuda").manual_seed(0)
    cache = torch.randint(0, 100, shape, generator=g, device="cuda").to(dtype)
    want = cache.clone().unsqueeze(0) if not layers else cache.clone()
    for a, b, n in PAIRS:
        if a >= 0 and b >= 0:
            if by_token:
                want[:, b, :, :n] = want[:, a, :, :n].clone()
            else:
                want[:, b] = want[:, a].clone()
    src, dst, n = (i32(list(x)) for x in zip(*PAIRS))
    ops.copy_pages(cache, src, dst, n if by_token else None, layers=layers)
    ops.check_status()
    assert torch.equal(cache, want.view(shape))


def test_copies_of_other_caches():
    g = torch.Generator("cuda").manual_seed(0)
    src, dst, n = (i32(list(x)) for x in zip(*PAIRS))
    rows = lambda *s: torch.randint(0, 100, s, generator=g, device="cuda").to(BF)  # noqa: E731
    pair, latent, quant = ops.KVPair(rows(14, 16, 2, 64), rows(14, 16, 2, 40)), ops.LatentKV(rows(14, 16, 1, 72), 64), ops.quant_kv_pool(14, 16, 2, 64, 32)
    quant.pool.copy_(torch.randint(0, 256, quant.pool.shape, generator=g, device="cuda"))
    for cache, tensors in ((pair, pair), (latent, (latent.pool,)), (quant, (quant.pool,))):
        want = [t.clone() for t in tensors]
        for a, b, m in PAIRS:
            for t in want:
                if a >= 0 and b >= 0:
                    t[b, :m if cache is not quant else 16] = t[a, :m if cache is not quant else 16].clone()
        ops.copy_pages(cache, src, dst, n)
        ops.check_status()
        assert all(torch.equal(a, b) for a, b in zip(tensors, want))
    before = latent.pool.clone()
    ops.copy_pages(latent, i32([14, 1]), i32([2, 100]))
    with pytest.raises(RuntimeError, match="index"):
        ops.check_status()
    assert torch.equal(before, latent.pool)
    for bad in (pair.k, before.transpose(0, 1), before[:, ::2]):        # tokens of pages that have no keys and values, caches in pieces
        with pytest.raises(ValueError):
            ops.copy_pages(bad, src, dst, n)
    with pytest.raises(ValueError):
        ops.copy_pages(pair, src, dst, n, layers=True)


# ---------------------------------------------------------------------------------------------------------- tables of a step
def _table_case(rng, R, W, page, beams):
    table, cached = [], []
    for _ in range(R // max(beams, 1)):
        n, common = rng.randrange(0, W * page), rng.randrange(0, W + 1)
        first = [rng.randrange(0, 500) for _ in range(W)]
        for _ in range(max(beams, 1)):
            table.append(first[:common] + [rng.randrange(0, 500) for _ in range(W - common)])
            cached.append(rng.choice([n, n, n, -1, rng.randrange(0, W * page)]))
    return table, cached


@pytest.mark.parametrize("R,W,page,beams", [(1, 1, 16, 1), (4, 17, 64, 4), (12, 40, 16, 3), (256, 9, 64, 8), (61, 300, 16, 0), (2, 2000, 64, 2), (1000, 3, 1, 5), (8192, 2, 128, 64), (5, 7, 48, 0)])
@pytest.mark.parametrize("ragged", [False, True])
def test_tables(R, W, page, beams, ragged):
    rng = random.Random(R * W + ragged)
    table, cached = _table_case(rng, R, W, page, beams)
    counts, T = None, 0
    if ragged:
        counts = [rng.choice([0, 1, 1, -3, rng.randrange(1, 2 * page)]) for _ in range(R)]
        counts = [min(n, W * page - max(c, 0)) for n, c in zip(counts, cached)]
        T = sum(max(n, 0) for n in counts) + 5
    got = ops.step_tables(i32(table), i32(cached), i32(counts) if ragged else None, page_size=page, beams=beams, tokens=T)
    ops.check_status()
    for g, w, name in zip(got, plain.tables(table, cached, counts, page, beams, R * W, T), ops.StepTables._fields):
        assert (g is None and w is None) or g.tolist() == w, name
    wide = torch.full((R, W + 5), 9, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + W] = i32(table)
    out = ops.StepTables(*(None if t is None else torch.full_like(t, 77) for t in got))
    again = ops.step_tables(wide[:, 2:2 + W], i32(cached), i32(counts) if ragged else None, page_size=page, beams=beams, tokens=T, out=out)
    assert again is out and all(a is None or torch.equal(a, b) for a, b in zip(got, out))


@pytest.mark.parametrize("entries,tokens", [(30, 1000), (1000, 100), (31, 57), (1, 1), (1000, 1)])
def test_tables_without_room(entries, tokens):
    rng = random.Random(entries + tokens)
    table, cached = _table_case(rng, 20, 6, 16, 0)
    counts = [min(rng.randrange(1, 20), 96 - max(c, 0)) for c in cached]
    for n in (counts, None):
        got = ops.step_tables(i32(table), i32(cached), None if n is None else i32(n), page_size=16, entries=entries, tokens=0 if n is None else tokens)
        want = plain.tables(table, cached, n, 16, 0, entries, tokens)
        for g, w, name in zip(got, want, ops.StepTables._fields):
            assert (g is None and w is None) or g.tolist() == w, name
        if n is not None or entries < 1000:
            with pytest.raises(RuntimeError, match="size beyond"):
                ops.check_status()
    ops.check_status()


def test_tables_of_rows_that_are_too_long():
    table = [[4, 5], [6, 7], [8, -1]]
    for cached, counts in (([32, 5, 16], None), ([31, 5, 2 ** 31 - 1], [2, 3, 4]), ([20, 5, 5], [2 ** 31 - 1, 3, 1])):
        got = ops.step_tables(i32(table), i32(cached), None if counts is None else i32(counts), page_size=16, tokens=0 if counts is None else 8, beams=3)
        with pytest.raises(RuntimeError, match="size beyond"):
            ops.check_status()
        for g, w, name in zip(got, plain.tables(table, cached, counts, 16, 3, 6, 8), ops.StepTables._fields):
            assert (g is None and w is None) or g.tolist() == w, name
    empty = ops.step_tables(i32([[0]])[:0], i32([0])[:0], i32([0])[:0], page_size=16, tokens=4)
    assert empty.indptr.tolist() == [0] and empty.slot.tolist() == [-1] * 4 and empty.pos.tolist() == [0] * 4


# ---------------------------------------------------------------------------------------------------------- attention
def _attend_case(seed, groups, beams, page, kvh, rep, dim, dtype):
    """groups: of each (full pages in common, tokens of every beam behind them)."""
    g = torch.Generator("cuda").manual_seed(seed)
    lists, lengths, shared, num = [], [], [], 0
    for common, tails in groups:
        first = list(range(num, num + common))
        num += common
        assert len(tails) == beams
        for t in tails:
            own = list(range(num, num + (-(-t // page) if t >= 0 else 0)))
            num += len(own)
            lists.append(first + own if t >= 0 else [])
            lengths.append(common * page + t if t >= 0 else 0)
        shared.append(common)
    perm = torch.randperm(num + 2, generator=torch.Generator().manual_seed(seed)).tolist()
    lists = [[perm[p] for p in x] for x in lists]
    kv = torch.randn(num + 2, 2, page, kvh, dim, generator=g, device="cuda").to(dtype)
    q = torch.randn(len(lists), (kvh * rep + 3) * dim, generator=g, device="cuda").to(dtype)
    indptr = [0]
    for x in lists:
        indptr.append(indptr[-1] + len(x))
    last = [(n - 1) % page + 1 if n else 0 for n in lengths]
    flat = [p for x in lists for p in x]
    return q, kv, i32(flat + [0]), i32(indptr), i32(last), i32(shared), lists, lengths


def _close(out, want, dtype, kv):
    """Weights (of sum one) enter the second product with half a step of the type, the output is rounded once: half a step each of the largest value's size.
    Scores of size s are off by s 2^-22 or so: within the slack."""
    half = torch.finfo(dtype).eps / 2
    top = kv[:, 1].double().nan_to_num(nan=0.0, posinf=0.0, neginf=0.0).clamp(-1e6, 1e6).abs().max().item()
    off = (out.double().cpu() - want).abs()
    assert (off <= half * (want.abs() + top * 1.25) + 1e-30).all(), (off.max().item(), half * top)


def _attend(case, beams, page, kvh, rep, dim, dtype, **more):
    q, kv, indices, indptr, last, shared, lists, lengths = case
    out = ops.attn_decode_beams(q, kv, indices, indptr, last, shared, beams=beams, q_heads=kvh * rep, kv_heads=kvh, head_dim=dim, page_size=page, **more)
    ops.check_status()
    want = plain.attend(q, kv, lists, lengths, kvh * rep, kvh, dim, scale=more.get("sm_scale"), cap=more.get("softcap", 0.0), sink=more.get("sink"))
    _close(out[:want.shape[0], :want.shape[1]], want, dtype, kv)
    return out


GROUPS = {
    "one token": (1, [(0, [1])]),
    "one page, one beam": (1, [(1, [0])]),
    "four beams": (4, [(15, [37, 37, 37, 37])]),
    "nothing in common": (3, [(0, [5, 70, 129]), (0, [64, 1, 1])]),
    "nothing behind": (2, [(3, [0, 0]), (1, [0, 0])]),
    "dead rows": (4, [(2, [3, -1, 0, 7]), (0, [-1, -1, -1, -1]), (0, [-1, 200, -1, 1]), (5, [-1, -1, -1, 64])]),
    "one dead row": (1, [(0, [-1])]),
    "many of unequal lengths": (5, [(i * 3 % 11, [(i * 7 + j * 13) % 90 for j in range(5)]) for i in range(1, 19)]),
    "long": (2, [(200, [1, 100]), (3, [2, 2])]),
    "sixteen beams": (16, [(9, list(range(16))), (2, [5] * 16)]),
}


@pytest.mark.parametrize("name", list(GROUPS))
@pytest.mark.parametrize("page,kvh,rep,dim,dtype", [(64, 2, 4, 128, BF), (16, 4, 4, 64, HF), (128, 1, 8, 128, HF), (16, 8, 1, 128, BF), (32, 2, 5, 64, BF)])
def test_attention(name, page, kvh, rep, dim, dtype):
    beams, groups = GROUPS[name]
    _attend(_attend_case(len(name), groups, beams, page, kvh, rep, dim, dtype), beams, page, kvh, rep, dim, dtype)


@pytest.mark.parametrize("rep,beams", [(1, 1), (3, 7), (7, 9), (8, 16), (12, 4), (16, 5), (2, 64), (5, 26)])
def test_attention_heads(rep, beams):
    groups = [(4, [(j * 5) % 40 for j in range(beams)]), (0, [j % 3 for j in range(beams)])]
    groups[1] = (0, [max(1, t) for t in groups[1][1]])
    for dim in (64, 128):
        _attend(_attend_case(rep, groups, beams, 16, 2, rep, dim, BF), beams, 16, 2, rep, dim, BF)


@pytest.mark.parametrize("rows,beams", [(1100, 5), (1030, 1), (2048, 64)])
def test_attention_of_many_rows(rows, beams):
    """More rows than one launch takes."""
    groups = [(i % 3, [1 + (i + j) % 20 if (i + j) % 7 else -1 for j in range(beams)]) for i in range(rows // beams)]
    _attend(_attend_case(rows, groups, beams, 16, 1, 2, 64, BF), beams, 16, 1, 2, 64, BF)


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_caps_sinks_scales(dim):
    case = _attend_case(5, GROUPS["dead rows"][1], 4, 16, 2, 4, dim, BF)
    sink = torch.randn(8, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(BF)
    for more in (dict(softcap=5.0), dict(sink=sink), dict(sink=sink, softcap=30.0, sm_scale=0.3), dict(sm_scale=0.0), dict(sm_scale=-0.2), dict(sink=torch.full_like(sink, -math.inf)),
                 dict(sink=torch.full_like(sink, 60.0))):
        _attend(case, 4, 16, 2, 4, dim, BF, **more)


def test_attention_of_large_scores():
    """One key takes all the weight, far above the others; scores of some hundred."""
    case = _attend_case(9, [(6, [40, 3]), (0, [17, 130])], 2, 16, 2, 4, 64, HF)
    case[0].mul_(8)
    case[1][:, 0].mul_(8)
    q, kv, indices, indptr, last, shared, lists, lengths = case
    out = ops.attn_decode_beams(q, kv, indices, indptr, last, shared, beams=2, q_heads=8, kv_heads=2, head_dim=64, page_size=16)
    want = plain.attend(q, kv, lists, lengths, 8, 2, 64)
    # scores of up to 800 are off by 800 x 2^-22, weights by twice that beside half a step of the type
    off = (out.double().cpu() - want).abs()
    assert (off <= (2.0 ** -11 + 1600 * 2.0 ** -22) * (want.abs() + 1.25 * kv[:, 1].abs().max().double().item())).all()


def test_attention_beside_attn_decode():
    """The same rows through attn_decode: both are within the bound of the plain form, and rows without pages are zeros in both."""
    case = _attend_case(5, GROUPS["many of unequal lengths"][1], 5, 64, 2, 4, 128, BF)
    q, kv, indices, indptr, last, shared, lists, lengths = case
    a = ops.attn_decode(q, kv, indices, indptr, last, q_heads=8, kv_heads=2, head_dim=128, page_size=64)
    b = _attend(case, 5, 64, 2, 4, 128, BF)
    assert (a.double() - b.double()).abs().max() <= 2 * 2.0 ** -8 * 2.25 * kv[:, 1].abs().max().double()


def test_attention_places():
    """Outputs with a pitch, rows behind the last left as they are, scratch of the size asked for, larger scratch for fewer rows."""
    beams, groups = GROUPS["dead rows"]
    case = _attend_case(2, groups, beams, 16, 2, 4, 64, BF)
    want = _attend(case, beams, 16, 2, 4, 64, BF)
    out = torch.full((20, 600), 7.0, dtype=BF, device="cuda")
    n = ops.attn_beams_workspace_bytes(64, beams, q_heads=8, kv_heads=2, head_dim=64, device="cuda")
    work = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    for _ in range(2):
        _attend(case, beams, 16, 2, 4, 64, BF, out=out[:, 8:], workspace=work)
        assert torch.equal(out[:16, 8:520], want)
        assert (out[16:] == 7).all() and (out[:, :8] == 7).all() and (out[:, 520:] == 7).all()
    with pytest.raises(ValueError):
        _attend(case, beams, 16, 2, 4, 64, BF, workspace=work[:0])
    with pytest.raises(ValueError):
        _attend(case, beams, 16, 2, 4, 64, BF, workspace=work[8:])


def test_attention_pages_that_there_are_not():
    case = list(_attend_case(2, [(2, [3, 5])], 2, 16, 2, 4, 64, BF))
    case[2] = case[2].clone()
    case[2][1] = 1 << 20
    case[2][2] = -5
    q, kv, indices, indptr, last, shared, _, _ = case
    ops.attn_decode_beams(q, kv, indices, indptr, last, shared, beams=2, q_heads=8, kv_heads=2, head_dim=64, page_size=16)
    with pytest.raises(RuntimeError, match="index"):
        ops.check_status()


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_attention_behind_a_row_s_end(dim, page):
    """Whatever a page holds behind its row's last token does not matter: numbers, infinities, NaN."""
    case = _attend_case(6, [(3, [1, 15, 17]), (0, [40, -1, 9])], 3, page, 2, 4, dim, BF)
    want = _attend(case, 3, page, 2, 4, dim, BF)
    for pages, n in zip(case[6], case[7]):
        if n % page:
            case[1][pages[-1], :, n % page:] = torch.tensor([math.nan, math.inf, -math.inf, 3e38], device="cuda").to(BF).repeat(dim // 4)
    assert torch.equal(_attend(case, 3, page, 2, 4, dim, BF), want)


def test_attention_captured():
    """A graph replayed with other lengths, tables and numbers of common pages than it was captured with."""
    a = _attend_case(3, [(5, [10, 20, 30, -1]), (1, [0, 1, 2, 3])], 4, 16, 2, 4, 64, BF)
    b = _attend_case(4, [(0, [1, 2, -1, 300]), (30, [9, 9, 9, 9])], 4, 16, 2, 4, 64, BF)
    room = max(a[1].shape[0], b[1].shape[0])
    q, kv = a[0].clone(), torch.zeros(room, *a[1].shape[1:], dtype=BF, device="cuda")
    kv[:a[1].shape[0]] = a[1]
    indices = torch.zeros(200, dtype=torch.int32, device="cuda")
    indices[:a[2].shape[0]] = a[2]
    indptr, last, shared = a[3].clone(), a[4].clone(), a[5].clone()
    more = dict(beams=4, q_heads=8, kv_heads=2, head_dim=64, page_size=16)
    out, graph = torch.zeros(8, 512, dtype=BF, device="cuda"), torch.cuda.CUDAGraph()
    ops.attn_decode_beams(q, kv, indices, indptr, last, shared, out=out, **more)
    with torch.cuda.graph(graph):
        ops.attn_decode_beams(q, kv, indices, indptr, last, shared, out=out, **more)
    for case in (a, b, a):
        q.copy_(case[0])
        kv[:case[1].shape[0]] = case[1]
        indices[:case[2].shape[0]] = case[2]
        indptr.copy_(case[3])
        last.copy_(case[4])
        shared.copy_(case[5])
        graph.replay()
        torch.cuda.synchronize()
        _close(out, plain.attend(case[0], case[1], case[6], case[7], 8, 2, 64), BF, case[1])
    ops.check_status()


# ---------------------------------------------------------------------------------------------------------- a step of a search
def test_a_step_captured():
    """Selection, tables, copies, the step's tables and attention in one graph, three steps long, beside the same in plain form."""
    Q, k, V, page, kvh, rep, dim, L, W, P = 2, 3, 500, 16, 2, 4, 64, 2, 6, 60
    g = torch.Generator("cuda").manual_seed(0)
    cache = torch.randn(L, P, 2, page, kvh, dim, generator=g, device="cuda").to(BF)
    pool = [list(range(0, 30)), list(range(59, 29, -1))]
    lens = [19, 47]
    table = [[pool[q][i] if i < -(-lens[q] // page) else -1 for i in range(W)] if b == 0 else [-1] * W for q in range(Q) for b in range(k)]
    cached = [lens[q] if b == 0 else -1 for q in range(Q) for b in range(k)]
    logits = torch.randn(Q * k, V, generator=g, device="cuda").to(BF)
    q = torch.randn(Q * k, kvh * rep * dim, generator=g, device="cuda").to(BF)
    tab, cac, scores = i32(table), i32(cached), torch.tensor([0.0 if b == 0 else -math.inf for _ in range(Q) for b in range(k)], device="cuda")
    out = torch.zeros(Q * k, kvh * rep * dim, dtype=BF, device="cuda")
    keep = {}

    def step():
        s = ops.beam_select(logits, scores, k, ended=None)
        f = ops.beam_fork(tab, cac, s.next_parent, i32_pool, page_size=page, num_pages=P)
        ops.copy_pages(cache, f.src, f.dst, f.tokens, layers=True)
        t = ops.step_tables(f.table, f.cached, page_size=page, beams=k)
        ops.attn_decode_beams(q, cache[1], t.indices, t.indptr, t.last_page_len, t.shared, beams=k, q_heads=kvh * rep, kv_heads=kvh, head_dim=dim, page_size=page, out=out)
        scores.copy_(s.next_score.view(-1))
        tab.copy_(f.table)
        cac.copy_(torch.where(f.cached >= 0, f.cached + 1, f.cached))
        keep.update(s=s, f=f, t=t)
    i32_pool = i32(pool)
    state = [t.clone() for t in (tab, cac, scores, cache)]
    step()
    torch.cuda.synchronize()
    for t, v in zip((tab, cac, scores, cache), state):
        t.copy_(v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    sc, kv = scores.tolist(), cache.cpu().clone()
    for i in range(3):
        logits.copy_(torch.randn(Q * k, V, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        ops.check_status()
        best, on, every = plain.select(logits, torch.tensor(sc), k, 2 * k, k)
        _same_selection(keep["s"], best, on, every, V)
        parents = [[b for _, b, _ in row] for row in on]
        table, cached, src, dst, n = plain.fork(table, cached, parents, pool, page, P)
        assert keep["f"].table.tolist() == table and keep["f"].cached.tolist() == cached
        for a, b, m in zip(src, dst, n):
            if a >= 0:
                kv[:, b, :, :m] = kv[:, a, :, :m]
        assert torch.equal(cache.cpu(), kv)
        fields = plain.tables(table, cached, None, page, k, Q * k * W, 0)
        for x, w in zip(keep["t"], fields):
            assert (x is None and w is None) or x.tolist() == w
        lengths = [c + 1 if c >= 0 else 0 for c in cached]
        _close(out, plain.attend(q, cache[1], [t[:-(-m // page)] for t, m in zip(table, lengths)], lengths, kvh * rep, kvh, dim), BF, cache)
        cached = [c + 1 if c >= 0 else c for c in cached]
        sc = scores.tolist()


def test_tables_of_pages_that_there_are_not():
    """A number whose slots do not fit into 32 bits gives none, and the status word says so; one without a page gives none."""
    table, cached = i32([[1 << 25, 5], [3, 1 << 30], [-1, -1], [7, 9]]), i32([7, 64, 3, 70])
    for counts, want in ((None, [-1, -1, -1, 9 * 64 + 6]), (i32([1, 0, 2, 3]), [-1, -1, -1, 9 * 64 + 6, 9 * 64 + 7, 9 * 64 + 8])):
        got = ops.step_tables(table, cached, counts, page_size=64, tokens=0 if counts is None else 6)
        with pytest.raises(RuntimeError, match="index out of range"):
            ops.check_status()
        assert got.slot.tolist() == want
    got = ops.step_tables(i32([[0]]), i32([(1 << 31) - 3]), page_size=(1 << 31) - 1)
    ops.check_status()
    assert got.indptr.tolist() == [0, 1] and got.last_page_len.tolist() == [(1 << 31) - 2] and got.slot.tolist() == [(1 << 31) - 3]


def test_no_requests():
    none = torch.empty(0, 3, dtype=torch.int32, device="cuda")
    got = ops.beam_fork(none, none[:, 0].contiguous(), torch.empty(0, 4, dtype=torch.int32, device="cuda"), none, page_size=16, num_pages=9)
    assert [tuple(t.shape) for t in got] == [(0, 3), (0,), (0,), (0,), (0,)]
    ops.check_status()


def test_select_rows_far_apart():
    """Rows whose elements are more than 2^32 behind the first one's."""
    pitch = (1 << 31) - 11
    room = torch.empty(2 * pitch + pitch // 2, dtype=BF, device="cuda")
    z = torch.as_strided(room, (3, 1003), (pitch, 1), 5)
    z.copy_(torch.randn(3, 1003, generator=torch.Generator("cuda").manual_seed(2), device="cuda"))
    _select(z, torch.zeros(3, device="cuda"), 3)


def test_pages_far_behind():
    """Attention over, and copies of, pages more than 2^32 elements into a cache."""
    page, kvh, rep, dim, beams = 64, 8, 2, 128, 3
    last = (1 << 32) // (2 * page * kvh * dim) + 40
    cache = torch.empty(last + 1, 2, page, kvh, dim, dtype=BF, device="cuda")
    g = torch.Generator("cuda").manual_seed(8)
    near = torch.randn(8, 2, page, kvh, dim, generator=g, device="cuda").to(BF)
    cache[:8] = near
    to = i32(list(range(last - 7, last + 1)))
    ops.copy_pages(cache, i32(list(range(8))), to)
    assert torch.equal(cache[-8:], near)
    q = torch.randn(beams, kvh * rep * dim, generator=g, device="cuda").to(BF)
    tables = [[0, 1, 2 + b] for b in range(beams)]
    indptr, tail, shared = i32([0, 3, 6, 9]), i32([5, 64, 17]), i32([2])
    more = dict(beams=beams, q_heads=kvh * rep, kv_heads=kvh, head_dim=dim, page_size=page)
    want = ops.attn_decode_beams(q, near, i32(sum(tables, [])), indptr, tail, shared, **more)
    got = ops.attn_decode_beams(q, cache, i32([last - 7 + p for t in tables for p in t]), indptr, tail, shared, **more)
    ops.check_status()
    assert torch.equal(got, want)
