"""A cache held in 4 bits on the GPU: numbers halfway between two codes, rows in runs of any length, portions over many rounds of blocks."""
import math

import pytest
import torch

from quant_kv_plain import attention, cache_at, read_back
from test_quant_kv_gpu import DEV, HALF, SIZES, filled, rows, stored, tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from blitz_scale_b200 import ops as o
    o.lib()
    return o


@pytest.fixture(autouse=True)
def _status(ops):
    yield
    ops.check_status()


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("dt,exponent", [(torch.bfloat16, e) for e in (-118, -105, -95, -60, 0, 50, 110)] + [(torch.float16, e) for e in (-12, -3, 0, 8)])
def test_numbers_halfway_between_two_codes(ops, group, dt, exponent):
    """Every scale of 8 bits, numbers at the middle of its steps and next to it: the code is the one that the definition's quotient rounds to."""
    D, g = 128, torch.Generator().manual_seed(exponent)
    s = (torch.arange(128, 256, dtype=torch.float64) / 128) * 2.0 ** exponent
    z = torch.randint(-12, 5, (128,), generator=g).double() * 2.0 ** exponent
    mid = (z[:, None] + s[:, None] * (torch.arange(15) + 0.5)).to(dt)
    step = (mid.view(torch.int16) + torch.randint(-1, 2, mid.shape, generator=g).to(torch.int16)).view(dt)
    ends = torch.stack([z, z + 15 * s], 1).to(dt)
    x = torch.cat([ends, mid, step], 1)                                    # 32 numbers of 128 groups
    x = x.view(128 * 32 // D, 1, D) if group == 32 else x.repeat(1, 4).view(128, 1, D)
    n = x.shape[0]
    cache = stored(ops, x, x, torch.arange(n), 1, D, group, 16, -(-n // 16))
    for held in cache_at(cache, torch.arange(n) // 16, torch.arange(n) % 16):
        assert torch.equal(held, read_back(x, group))


@pytest.mark.parametrize("D,group", SIZES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("longest", [3, 9, 40])
def test_rows_in_runs(ops, D, group, dt, longest):
    """Runs of rows that follow one another in a page, from any offset on, and rows that nobody wants among them."""
    H, page, T = 3, 64, 203
    g = torch.Generator().manual_seed(longest)
    starts, slot = torch.randperm(T, generator=g) * 64, []
    while len(slot) < T:
        n = min(int(torch.randint(1, longest + 1, (1,), generator=g)), 64, T - len(slot))
        first = int(torch.randint(0, 65 - n, (1,), generator=g))
        slot += [int(starts[len(slot)]) + first + i for i in range(n)]
    slot = torch.tensor(slot)
    want = torch.rand(T, generator=g) > 0.1
    k, v = rows(T, H, D, dt, 5), rows(T, H, D, dt, 6)
    cache = stored(ops, k, v, torch.where(want, slot, -1), H, D, group, page, T)
    held = cache_at(cache, slot // page, slot % page)
    out = [torch.full((T, H, D), 3.0, dtype=dt, device=DEV) for _ in range(2)]
    some = torch.rand(T, generator=g) > 0.1
    ops.quant_kv_load(cache, torch.where(some, slot, -7).to(torch.int32).to(DEV), k=out[0], v=out[1])
    for x, h, y in zip((k, v), held, out):
        assert torch.equal(h[want], read_back(x, group)[want]) and not h[~want].any()
        y = y.cpu().double()
        # (rounded once from 32 bits)
        assert ((y - h).abs() <= (HALF[dt] + 2.0 ** -23) * h.abs() + 2.0 ** -25)[some].all()
        assert (y[~some] == 3.0).all()
    assert int((cache.pool != 0).any(-1).sum()) <= int(want.sum()) * H


# sequences of a head that a block has to itself, more of them than blocks, some that are cut; empty ones among them
WHOLE = [([32 * 37] * 18, 8), ([900 + 31 * i for i in range(18)] + [0], 8), ([0, 0, 1], 1), ([1] * 37, 4), ([200 - 3 * i for i in range(61)], 8),
         ([0, 33] * 130 + [1], 4), ([3 * i for i in range(200)], 2), ([700] * 20, 8), ([5000] + [20] * 40, 2)]


@pytest.mark.parametrize("case", range(len(WHOLE)))
@pytest.mark.parametrize("window", [0, 70])
def test_blocks_of_whole_sequences(ops, case, window):
    (lens, H), rep, D, group, page, dt = WHOLE[case], 4, 64, 32, 16, torch.float16
    cache, table, indptr, last, kept = filled(ops, lens, H, D, group, page, dt, 10 * case)
    q = torch.randn(len(lens), rep * H, D, generator=torch.Generator().manual_seed(case)).to(dt)
    got = ops.attn_decode(q.flatten(1).to(DEV), cache, table, indptr, last, q_heads=rep * H, kv_heads=H, head_dim=D, page_size=page, window=window)
    got = got.cpu().double().view(len(lens), rep * H, D)
    for s, n in enumerate(lens):
        if n == 0:
            assert not got[s].any()
            continue
        k, v, ks, kz, vs = kept[s]
        at = torch.tensor([n - 1])
        want = attention(q[s:s + 1], k, v, at, scale=D ** -0.5, window=window)
        spread = attention(q[s:s + 1], k, 8 * vs.repeat_interleave(group, -1), at, scale=D ** -0.5, window=window)[0]
        step = 2.0 ** -11 + 2.0 ** -15 + n / 16 * 2.0 ** -22        # (as for single tokens in general)
        tol = tolerance(q[s:s + 1], kept[s], D ** -0.5, want, spread, step, dt, group) + n * 2.0 ** -28 * vs.max()
        assert ((got[s] - want[0][0]).abs() <= tol[0]).all(), (s, n)


def test_portions_of_many_rounds(ops):
    """More work than blocks, tiles of one row, of all rows and of none, rows of queries 2^-40 to 2^2 as large as others."""
    n, Q, H, D, group, page, dt = [1, 128, 129, 256, 257, 400, 700, 511], 32, 8, 128, 64, 64, torch.bfloat16
    lens = [m + 37 * i for i, m in enumerate(n)]
    cache, table, _, _, kept = filled(ops, lens, H, D, group, page, dt, 77)
    g = torch.Generator().manual_seed(8)
    q = (torch.randn(sum(n), Q, D, generator=g) * 2.0 ** torch.randint(-40, 3, (sum(n), Q, 1), generator=g)).to(dt)
    more = dict(q_heads=Q, kv_heads=H, head_dim=D, page_size=page)
    work = ops.prefill_work_list(n, lens, page, DEV)
    run = lambda q: ops.attn_prefill_paged(q.flatten(1).to(DEV), cache, table, work, **more).cpu().view(-1, Q, D)  # noqa: E731
    got, row = run(q), 0
    for s, b in enumerate(n):
        k, v, ks, kz, vs = kept[s]
        x = q[row:row + b]
        want = attention(x, k, v, torch.arange(lens[s] - b, lens[s]), scale=D ** -0.5)
        half = 2.0 ** -11
        tol = tolerance(x, kept[s], D ** -0.5, want, want[1], half, dt, group, value_step=half)
        # (beside the largest key of any sequence's head and of the row's own queries, below 2^-14 of them in steps of 2^-24)
        largest = max(float(m[0].abs().max()) for m in kept)
        floor = 2.0 ** -24 * largest * x.double().abs().sum(-1) * D ** -0.5 + 2.0 ** -24 * x.double().abs().amax(-1) * D * largest * D ** -0.5
        tol = tol + torch.expm1(2 * floor)[..., None] * want[1] + 2.0 ** -24 * max(float(m[1].abs().max()) for m in kept)
        assert ((got[row:row + b].double() - want[0]).abs() <= tol).all(), s
        row += b
    # a row that is no number, or far larger, changes no other
    other = q.clone()
    for i, x in ((0, math.nan), (140, math.inf), (141, 1e30), (900, -math.inf), (sum(n) - 1, math.nan)):
        other[i, 5] = x
    keep = torch.ones(sum(n), Q, dtype=torch.bool)
    keep[[0, 140, 141, 900, sum(n) - 1], 5] = False
    again = run(other)
    assert torch.equal(again[keep], got[keep]) and again[0, 5].isnan().all() and again[-1, 5].isnan().all()


def test_chunks_that_do_not_fit_are_refused(ops):
    """Chunks are counted in 32 bits: the table's length says how many there can be."""
    cache = ops.quant_kv_pool(1, 1 << 16, 1, 64, 64)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    q = torch.zeros(1, 8 * 64, dtype=torch.bfloat16, device=DEV)
    table = torch.zeros(1 << 20, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="chunks"):
        ops.attn_decode(q, cache, table, t([0, 1]), t([1]), q_heads=8, kv_heads=1, head_dim=64, page_size=1 << 16)


def test_pages_that_there_are_not(ops):
    """A page or slot behind the cache is an error that the host reads; nothing is written for it, and rows beside it are what they were."""
    H, D, group, page, n = 2, 64, 32, 16, 40
    cache, table, indptr, last, _ = filled(ops, [n], H, D, group, page, torch.bfloat16, 9)
    pages, t = cache.pool.shape[0], lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    k, before = rows(3, H, D, torch.bfloat16, 10).to(DEV), cache.pool.clone()
    qkv = torch.zeros(2, 4 * H * D, dtype=torch.bfloat16, device=DEV)
    more = dict(q_heads=2 * H, kv_heads=H, head_dim=D, page_size=page)
    q = torch.ones(n, 2 * H * D, dtype=torch.bfloat16, device=DEV)
    out = torch.full((3, 2, page, H, D), 5.0, dtype=torch.bfloat16, device=DEV)
    load = torch.full((3, H, D), 5.0, dtype=torch.bfloat16, device=DEV)
    far = [pages * page, (1 << 31) - 1]
    calls = [lambda: ops.quant_kv_store(k[:2], k[:2], t(far), cache), lambda: ops.quant_kv_load(cache, t([far[0], 1, far[1]]), k=load, v=load.clone()),
             lambda: ops.quant_kv_pages(cache, t([pages, 0, -1]), out=out), lambda: ops.rope_kv_store(qkv, t([0, 1]), t(far), cache, rope_theta=1e4, **more)]
    for bad in (pages, -1, 1 << 30):
        wrong = table.clone()
        wrong[1] = bad
        calls += [lambda w=wrong: ops.attn_decode(q[:1], cache, w, indptr, last, **more),
                  lambda w=wrong: ops.attn_prefill_paged(q, cache, w, ops.prefill_work_list([n], [n], page, DEV), **more)]
    for i, call in enumerate(calls):
        call()
        with pytest.raises(RuntimeError):
            ops.check_status()
        assert torch.equal(cache.pool, before), i
    assert (out[[0, 2]] == 5.0).all() and torch.equal(out[1, 0].flatten(0, 1), ops.quant_kv_load(cache, torch.arange(page, dtype=torch.int32, device=DEV))[0].flatten(0, 1))
    assert (load[[0, 2]] == 5.0).all() and not (load[1] == 5.0).all()
