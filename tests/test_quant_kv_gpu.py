"""A cache held in 4 bits on the GPU: what is written and read back, attention of single tokens and of portions, against 64 bits."""
import math

import pytest
import torch

from quant_kv_plain import attention, cache_at, quantised, read_back, values

pytestmark = pytest.mark.gpu
DEV = "cuda"
SIZES = [(128, 32), (128, 64), (128, 128), (64, 32), (64, 64)]
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}       # half a step, relative


@pytest.fixture(scope="module")
def ops():
    from blitz_scale_b200 import ops as o
    o.lib()
    return o


@pytest.fixture(autouse=True)
def _status(ops):
    yield
    ops.check_status()


def rows(n, H, D, dt, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, H, D, generator=g)
    x[:, :, ::29] *= 5.0
    return (x + torch.randn(1, H, D, generator=g)).to(dt)


def stored(ops, k, v, slot, H, D, group, page, pages, pitch=0):
    """A cache with rows k, v at their slots, which come with a pitch of `pitch` more elements."""
    cache = ops.quant_kv_pool(pages, page, H, D, group)
    wide = lambda x: torch.cat([x.flatten(1), torch.full((x.shape[0], pitch), 7.0, dtype=x.dtype)], 1).to(DEV)[:, :H * D]  # noqa: E731
    ops.quant_kv_store(wide(k), wide(v), slot.to(torch.int32).to(DEV), cache)
    return cache


@pytest.mark.parametrize("D,group", SIZES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,page,T", [(1, 16, 1), (2, 64, 3), (8, 64, 129), (5, 128, 333), (3, 16, 67)])
def test_codes_and_what_is_read_back(ops, D, group, dt, H, page, T):
    """Every code, scale and offset is the definition's; rows read back are those values, rounded once."""
    pages = -(-T // page) + 3
    g = torch.Generator().manual_seed(T)
    slot = torch.randperm(pages * page, generator=g)[:T]
    k, v = rows(T, H, D, dt, 1), rows(T, H, D, dt, 2)
    cache = stored(ops, k, v, slot, H, D, group, page, pages, pitch=16)
    held = cache_at(cache, slot // page, slot % page)
    got = ops.quant_kv_load(cache, slot.to(torch.int32).to(DEV), dtype=dt)
    for x, h, y in zip((k, v), held, got):
        assert torch.equal(h, read_back(x, group))
        # (z + s c has up to 8 + 12 significant bits in 32: a fused sum rounds once, to 24, then to 16)
        assert ((y.cpu().double() - h).abs() <= (HALF[dt] + 2.0 ** -23) * h.abs() + 2.0 ** -25).all()
    # nothing else was written
    free = torch.ones(pages * page, dtype=torch.bool)
    free[slot] = False
    rest = free.nonzero().flatten()
    for h in cache_at(cache, rest // page, rest % page):
        assert not h.any()


@pytest.mark.parametrize("D,group", [(128, 32), (128, 128), (64, 64)])
@pytest.mark.parametrize("page", [16, 64])
def test_pages_read_back_are_the_rows(ops, D, group, page):
    H, n = 3, 5
    cache = ops.quant_kv_pool(n + 2, page, H, D, group)
    cache.pool.copy_(torch.randint(0, 256, cache.pool.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(1)))
    # scales and offsets that are numbers
    codes, part = 8 * D, cache.pool.shape[3] // 2
    for at in (codes, part + codes):
        w = torch.randn(*cache.pool.shape[:3], 32 * (D // group), generator=torch.Generator().manual_seed(at)).to(torch.bfloat16)
        cache.pool[..., at:at + 64 * (D // group)] = w.view(torch.uint8).view(*cache.pool.shape[:3], -1).to(DEV)
    pages = torch.tensor([4, 0, n + 1, 4, 2], dtype=torch.int32, device=DEV)
    whole = ops.quant_kv_pages(cache, pages)
    slot = (pages.long()[:, None] * page + torch.arange(page, device=DEV)).flatten().to(torch.int32)
    k, v = ops.quant_kv_load(cache, slot)
    assert torch.equal(whole[:, 0].reshape(-1, H, D), k) and torch.equal(whole[:, 1].reshape(-1, H, D), v)


def test_rows_without_a_slot_and_rows_in_slots_of_others(ops):
    cache = ops.quant_kv_pool(3, 16, 2, 64, 32)
    k, v = rows(4, 2, 64, torch.bfloat16, 3).to(DEV), rows(4, 2, 64, torch.bfloat16, 4).to(DEV)
    ops.quant_kv_store(k.flatten(1), v, torch.tensor([17, -1, 18, -1], dtype=torch.int32, device=DEV), cache)
    before = cache.pool.clone()
    k1, v1 = ops.quant_kv_load(cache, torch.tensor([17, 18], dtype=torch.int32, device=DEV))
    ops.quant_kv_store(k[1:2], v[1:2], torch.tensor([19], dtype=torch.int32, device=DEV), cache)     # the same word of the values' codes
    k2, v2 = ops.quant_kv_load(cache, torch.tensor([17, 18], dtype=torch.int32, device=DEV))
    assert torch.equal(k1, k2) and torch.equal(v1, v2) and not torch.equal(before, cache.pool)
    out = torch.full((3, 2, 64), 5.0, dtype=torch.bfloat16, device=DEV)
    ops.quant_kv_load(cache, torch.tensor([-1, 17, -1], dtype=torch.int32, device=DEV), k=out, v=out.clone())
    assert (out[[0, 2]] == 5.0).all() and torch.equal(out[1], k1[0])
    ops.quant_kv_store(k[:0], v[:0], torch.zeros(0, dtype=torch.int32, device=DEV), cache)


def test_groups_of_one_number_extremes_and_what_is_no_number(ops):
    cache = ops.quant_kv_pool(1, 16, 1, 64, 32)
    k = torch.zeros(7, 1, 64, dtype=torch.bfloat16)
    k[0] = 3.7                                     # a range of zero
    k[1, 0, :32] = torch.finfo(torch.bfloat16).max  # the largest number beside its negative: wider than fp32
    k[1, 0, 1] = -torch.finfo(torch.bfloat16).max
    k[2, 0, 40] = math.inf
    k[3, 0, 3] = math.nan
    k[4, 0, :32] = torch.arange(32) * 2.0 ** -133   # the smallest numbers there are
    k[5, 0, 32:] = torch.linspace(0, 15, 32)        # ties
    k[6, 0, :32] = torch.linspace(1.0e38, 2.9e38, 32)
    slot = torch.arange(7, dtype=torch.int32, device=DEV)
    ops.quant_kv_store(k[:, 0].to(DEV), k.to(DEV), slot, cache)
    for y in ops.quant_kv_load(cache, slot):
        y = y.cpu()
        assert torch.equal(y[0], k[0])
        assert y[1, 0, :32].isnan().all() and not y[1, 0, 32:].any()
        assert y[2, 0, 32:].isnan().all() and not y[2, 0, :32].any()
        assert y[3, 0, :32].isnan().all() and not y[3, 0, 32:].any()
        # (bf16 has whole multiples of 2^-133 there: s = 3 of them for a range of 31)
        assert ((y[4].double() - k[4].double()).abs() <= 2 * 2.0 ** -133).all()
        for r in (5, 6):
            want = read_back(k[r], 32)
            assert ((y[r].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -23) * want.abs()).all()
    half = torch.full((1, 64), 65504.0, dtype=torch.float16, device=DEV)
    half[0, 0] = -65504.0
    ops.quant_kv_store(half, half, slot[:1], cache)
    assert torch.equal(ops.quant_kv_load(cache, slot[:1], dtype=torch.float16)[0].view(1, 64).abs(), half.abs())


# ---------------------------------------------------------------------------------------------------- attention
def filled(ops, lens, H, D, group, page, dt, seed, behind=255):
    """(cache, page table, indptr, last page lengths, keys and values of every sequence in 64 bits, what their codes span)"""
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lens]
    table = torch.randperm(sum(used) + 3, generator=g)[:sum(used)]
    cache = ops.quant_kv_pool(sum(used) + 3, page, H, D, group)
    cache.pool.fill_(behind)            # 255: what no sequence holds is no number
    kept, at = [], 0
    for s, n in enumerate(lens):
        k, v = rows(n, H, D, dt, seed + 2 * s), rows(n, H, D, dt, seed + 2 * s + 1)
        j = torch.arange(n)
        slot = table[at + j // page] * page + j % page if n else j
        at += used[s]
        ops.quant_kv_store(k.flatten(1).to(DEV), v.flatten(1).to(DEV), slot.to(torch.int32).to(DEV), cache)
        (kc, ks, kz), (vc, vs, vz) = quantised(k, group), quantised(v, group)
        kept.append((values(kc, ks, kz, group), values(vc, vs, vz, group), ks, kz, vs))
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    indptr = [0]
    for n in used:
        indptr.append(indptr[-1] + n)
    return cache, table.to(torch.int32).to(DEV), t(indptr), t([(n - 1) % page + 1 if n else 0 for n in lens]), kept


def tolerance(q, kept, scale, want, spread, weight_step, dt, group, value_step=0.0):
    """What arithmetic allows for rows q [n, heads, D] of a sequence.  Weights: a score is a sum of products that are exact in 32 bits, of
    codes that enter as numbers whose leading bit may be ten places up (a sum of `group` of them is off by less than 2^-22 of 1040 |q|
    each), times s, and
    of offsets z times sums of q that are held in 16 bits: |error| <= scale sum_g (2^-12 s_g + 2^-16 |z_g|) sum |q|, and 2^-20 of
    the score for the rest.  Every weight, and their sum, is off by that factor at most, so twice.  Then the rounding of a weight times its
    scale (`weight_step`) times codes between -8 and 7, of values where they are read back (`value_step`), and of the output."""
    k, v, ks, kz, vs = kept
    rep = q.shape[1] // k.shape[1]
    per_group = (2.0 ** -12 * ks + 2.0 ** -16 * kz.abs()).amax(0).repeat_interleave(rep, 0)         # [heads, groups]
    qs = q.double().abs().unflatten(-1, (-1, group)).sum(-1)
    off = scale * (qs * per_group).sum(-1) + 2.0 ** -20 * want[2] + value_step * scale * (q.double().abs() * k.abs().amax(0).repeat_interleave(rep, 0)).sum(-1)
    return (torch.expm1(2 * off)[..., None] * want[1] + weight_step * spread + value_step * want[1] + (HALF[dt] + 2.0 ** -20) * want[0].abs() + 1e-7)


# lengths (0: a row of padding), query and KV heads, head size, group, page, more
DECODE = [
    ([977], 32, 8, 128, 32, 64, {}),
    ([1], 8, 1, 64, 32, 16, {}),
    ([0, 0, 5, 0], 8, 2, 64, 64, 64, {}),
    ([3, 700, 64, 65, 0, 2049, 1, 16, 17], 16, 4, 128, 32, 64, {}),
    ([31, 33, 47, 15, 128, 127], 4, 4, 128, 64, 16, {}),
    ([513] * 40 + [7, 3000], 8, 8, 128, 128, 64, {}),
    ([600, 33, 1500], 12, 1, 64, 64, 32, {"sink": True, "window": 300, "keep_first": 70, "softcap": 20.0}),
    ([600, 33, 1500, 0], 8, 2, 128, 32, 128, {"window": 1}),
    ([900, 130, 1], 10, 2, 64, 32, 64, {"window": 64, "keep_first": 1}),
    ([30 + 7 * i for i in range(64)], 4, 2, 64, 64, 64, {"sink": True}),
    ([257, 5], 20, 1, 128, 128, 256, {"softcap": 5.0}),
    ([100] * 3, 16, 16, 128, 64, 64, {"keep_first": 5}),
]


@pytest.mark.parametrize("case", range(len(DECODE)))
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("splits", [0, 1])
def test_decode(ops, case, dt, splits):
    lens, Q, H, D, group, page, opts = DECODE[case]
    opts = dict(opts)
    cache, table, indptr, last, kept = filled(ops, lens, H, D, group, page, dt, 100 * case)
    g = torch.Generator().manual_seed(case)
    q = torch.randn(len(lens), Q, D, generator=g).to(dt)
    if opts.pop("sink", False):
        opts["sink"] = torch.randn(Q, generator=g).to(dt)
    scale = 1.2 * D ** -0.5
    wide = torch.cat([q.flatten(1), torch.full((len(lens), 64), math.nan, dtype=dt)], 1).to(DEV)        # columns of a fused projection
    dev = {n: x.to(DEV) if isinstance(x, torch.Tensor) else x for n, x in opts.items()}
    out = torch.full((len(lens) + 1, Q * D + 8), 9.0, dtype=dt, device=DEV)
    ops.attn_decode(wide, cache, table, indptr, last, q_heads=Q, kv_heads=H, head_dim=D, page_size=page, num_splits=splits, sm_scale=scale,
                    out=out[:len(lens), :Q * D], **dev)
    assert (out[len(lens)] == 9.0).all() and (out[:, Q * D:] == 9.0).all()
    got = out[:len(lens), :Q * D].cpu().double().view(len(lens), Q, D)
    for s, n in enumerate(lens):
        if n == 0:
            assert not got[s].any()
            continue
        k, v, ks, kz, vs = kept[s]
        at = torch.tensor([n - 1])
        want = attention(q[s:s + 1], k, v, at, scale=scale, **opts)
        spread = attention(q[s:s + 1], k, 8 * vs.repeat_interleave(group, -1), at, scale=scale, **opts)[0]
        # weights times scales in fp16 (below 2^-14 in steps of 2^-24, where the largest scale is at 2^6 at least); their products with codes (as
        # if up to 1039), 16 tokens at a time, and with 8, are sums in 32 bits beside the output so far: 2^-22 of their parts
        step = 2.0 ** -11 + 2.0 ** -15 + n / 16 * 2.0 ** -22
        tol = tolerance(q[s:s + 1], kept[s], scale, want, spread, step, dt, group) + n * 2.0 ** -28 * vs.max()
        worst = ((got[s] - want[0][0]).abs() / tol[0]).max().item()
        assert worst <= 1, (s, n, worst)


@pytest.mark.parametrize("rep", [4, 8])
@pytest.mark.parametrize("scale", [-0.11, 0.0, 0.07])
@pytest.mark.parametrize("softcap", [0.0, 3.0])
def test_decode_scales(ops, rep, scale, softcap):
    """A factor of either sign, or zero; queries and factor times powers of two that cancel change no bit."""
    lens, H, D, group, dt = [300, 1, 2000], 2, 128, 32, torch.bfloat16
    cache, table, indptr, last, kept = filled(ops, lens, H, D, group, 64, dt, 7)
    q = torch.randn(len(lens), rep * H, D, generator=torch.Generator().manual_seed(3)).to(dt)
    run = lambda q, scale: ops.attn_decode(q.flatten(1).to(DEV), cache, table, indptr, last, q_heads=rep * H, kv_heads=H, head_dim=D, page_size=64,
                                           num_splits=0, sm_scale=scale, softcap=softcap).cpu()
    got = run(q, scale)
    for s, n in enumerate(lens):
        k, v, ks, kz, vs = kept[s]
        want = attention(q[s:s + 1], k, v, torch.tensor([n - 1]), scale=scale, softcap=softcap)
        spread = attention(q[s:s + 1], k, 8 * vs.repeat_interleave(group, -1), torch.tensor([n - 1]), scale=scale, softcap=softcap)[0]
        step = 2.0 ** -11 + 2.0 ** -15 + n / 16 * 2.0 ** -22
        tol = tolerance(q[s:s + 1], kept[s], abs(scale), want, spread, step, dt, group) + n * 2.0 ** -28 * vs.max()
        assert ((got[s].double().view(-1, D) - want[0][0]).abs() <= tol[0]).all(), (s, n)
    for e in (-100, -30, 30, 100):
        assert torch.equal(run((q.float() * 2.0 ** e).to(dt), scale * 2.0 ** -e), got), e


# (tokens cached before, rows) of every sequence
PORTIONS = [
    ([(0, 1)], 4, 2, 128, 32, 64, {}),
    ([(0, 117), (33, 5)], 8, 2, 128, 64, 64, {}),
    ([(300, 260), (0, 63), (5, 1)], 4, 4, 64, 32, 16, {}),
    ([(70, 300)], 8, 1, 64, 64, 64, {"window": 100, "keep_first": 3, "sink": True}),
    ([(0, 200), (129, 129)], 4, 1, 128, 128, 32, {"softcap": 15.0}),
]


@pytest.mark.parametrize("case", range(len(PORTIONS)))
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_portions(ops, case, dt):
    seqs, Q, H, D, group, page, opts = PORTIONS[case]
    opts = dict(opts)
    lens, n = [a + b for a, b in seqs], [b for _, b in seqs]
    cache, table, _, _, kept = filled(ops, lens, H, D, group, page, dt, 1000 + case)
    g = torch.Generator().manual_seed(case)
    q = torch.randn(sum(n), Q, D, generator=g).to(dt)
    if opts.pop("sink", False):
        opts["sink"] = torch.randn(Q, generator=g).to(dt)
    dev = {m: x.to(DEV) if isinstance(x, torch.Tensor) else x for m, x in opts.items()}
    work = ops.prefill_work_list(n, lens, page, DEV)
    got = ops.attn_prefill_paged(q.flatten(1).to(DEV), cache, table, work, q_heads=Q, kv_heads=H, head_dim=D, page_size=page, **dev)
    got = got.cpu().double().view(-1, Q, D)
    row = 0
    for s, (a, b) in enumerate(seqs):
        k, v, ks, kz, vs = kept[s]
        x, at = q[row:row + b], torch.arange(a, a + b)
        want = attention(x, k, v, at, scale=D ** -0.5, **opts)
        # keys and values rounded to fp16, beside the largest of their head (below 2^-14 of it, in steps of 2^-24), and the weights
        half = 2.0 ** -11
        tol = tolerance(x, kept[s], D ** -0.5, want, want[1], half, dt, group, value_step=half)
        floor = 2.0 ** -24 * k.abs().amax() * x.double().abs().sum(-1) * D ** -0.5
        tol = tol + torch.expm1(2 * floor)[..., None] * want[1] + 2.0 ** -24 * v.abs().amax()
        worst = ((got[row:row + b] - want[0]).abs() / tol).max().item()
        assert worst <= 1, (s, worst)
        row += b
