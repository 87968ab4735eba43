"""Attention of portions over a 4-bit cache: keys and values of very different sizes, in one pass, one sequence, one head."""
import pytest
import torch

from quant_kv_plain import attention, quantised, values
from test_quant_kv_gpu import DEV, rows, tolerance

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


class Pass:
    """Rows of sequences [(tokens before, rows)], whose keys and values [tokens, heads, dim] are given; `lead` pages of nobody in front."""

    def __init__(self, ops, seqs, kv, q, group, page, lead=0, **opts):
        self.ops, self.group, self.page, self.lead, self.q = ops, group, page, lead, q
        self.H, self.D = kv[0][0].shape[1:]
        self.opts = {n: x.to(DEV) if isinstance(x, torch.Tensor) else x for n, x in opts.items()}
        self.lens, self.rows = [a + b for a, b in seqs], [b for _, b in seqs]
        used = [-(-n // page) for n in self.lens]
        g = torch.Generator().manual_seed(len(seqs))
        self.table = torch.randperm(sum(used) + 3, generator=g)[:sum(used)]
        self.cache = ops.quant_kv_pool(sum(used) + 3, page, self.H, self.D, group)
        self.cache.pool.fill_(255)
        at = 0
        for n, u, (k, v) in zip(self.lens, used, kv):
            j = torch.arange(n)
            slot = (self.table[at + j // page] * page + j % page).to(torch.int32).to(DEV)
            ops.quant_kv_store(k.flatten(1).to(DEV), v.flatten(1).to(DEV), slot, self.cache)
            at += u

    def run(self, cache=None):
        Q = self.q.shape[1]
        pages = torch.cat([torch.zeros(self.lead, dtype=torch.long), self.table]).to(torch.int32).to(DEV)
        work = self.ops.prefill_work_list([1] * bool(self.lead) + self.rows, [self.lead * self.page] * bool(self.lead) + self.lens, self.page, DEV,
                                          skip=int(self.lead > 0))
        x = torch.cat([torch.zeros(int(self.lead > 0), Q, self.D, dtype=self.q.dtype), self.q]).flatten(1).to(DEV)
        more = dict(skip_pages=self.lead) if cache is None else {}
        out = self.ops.attn_prefill_paged(x, self.cache if cache is None else cache, pages, work, q_heads=Q, kv_heads=self.H, head_dim=self.D,
                                          page_size=self.page, **more, **self.opts)
        return out[int(self.lead > 0):].cpu().view(-1, Q, self.D)

    def run_16_bit(self):
        """The same over a cache in bf16."""
        cache = self.ops.quant_kv_pages(self.cache, torch.arange(self.cache.pool.shape[0], dtype=torch.int32, device=DEV))
        # (what no sequence holds is no number, and the kernel of a 16-bit cache wants numbers)
        return self.run(torch.nan_to_num(cache, nan=0.0))

    def of(self, s):
        first = sum(self.rows[:s])
        return slice(first, first + self.rows[s])


def _kv(lens, H, D, seed):
    return [(rows(n, H, D, torch.bfloat16, seed + 2 * s), rows(n, H, D, torch.bfloat16, seed + 2 * s + 1)) for s, n in enumerate(lens)]


SHAPES = [([(0, 300), (170, 90), (65, 400)], 8, 2, 128, 32, 64, 0, {}),
          ([(0, 70), (3, 500), (0, 1)], 4, 4, 64, 64, 16, 5, {"window": 150, "keep_first": 2}),
          ([(20, 20), (0, 410), (128, 128)], 6, 2, 128, 128, 128, 1, {"softcap": 30.0})]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("huge", [1e30, 3e5, -1e20])
def test_large_numbers_of_a_sequence_leave_others_and_earlier_rows_alone(ops, shape, huge):
    seqs, Q, H, D, group, page, lead, opts = SHAPES[shape]
    kv = _kv([a + b for a, b in seqs], H, D, 50 * shape)
    g = torch.Generator().manual_seed(shape)
    q = torch.randn(sum(b for _, b in seqs), Q, D, generator=g).to(torch.bfloat16)
    plain = Pass(ops, seqs, kv, q, group, page, lead, **opts).run()
    at = seqs[1][0] + seqs[1][1] // 2          # a token that half of the rows see
    k, v = (x.clone() for x in kv[1])
    k[at, 0, D // 2], v[at, 0, 5] = huge, -huge
    p = Pass(ops, seqs, [kv[0], (k, v), kv[2]], q, group, page, lead, **opts)
    got = p.run()
    for s in (0, 2):
        assert torch.equal(got[p.of(s)], plain[p.of(s)])
    mine, rep = got[p.of(1)], Q // H
    assert torch.equal(mine[:, rep:], plain[p.of(1)][:, rep:])         # its other heads
    # the head's rows: as over a cache in bf16 (no numbers where a score passes 2^31, here and there), and those before the token as right as there
    assert torch.allclose(mine[:, :rep], p.run_16_bit()[p.of(1)][:, :rep], rtol=0, atol=0, equal_nan=True)
    first, n = seqs[1][0], at - seqs[1][0]
    (kc, ks, kz), (vc, vs, vz) = quantised(k[:at], group), quantised(v[:at], group)
    kept = (values(kc, ks, kz, group), values(vc, vs, vz, group), ks, kz, vs)
    x, half = q[p.of(1)][:n], 2.0 ** -8
    want = attention(x, kept[0], kept[1], torch.arange(first, at), scale=D ** -0.5, **opts)
    tol = tolerance(x, kept, D ** -0.5, want, want[1], half, torch.bfloat16, group, value_step=half)
    assert ((mine[:n].double() - want[0]).abs() <= tol).all()


@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_sequences_of_any_size_in_one_pass(ops, shape):
    """Keys times powers of two that the sequence's queries take back, and values times powers of two: outputs times those, bit for bit."""
    seqs, Q, H, D, group, page, lead, opts = SHAPES[shape]
    kv = _kv([a + b for a, b in seqs], H, D, 50 * shape + 9)
    q = torch.randn(sum(b for _, b in seqs), Q, D, generator=torch.Generator().manual_seed(shape)).to(torch.bfloat16)
    plain = Pass(ops, seqs, kv, q, group, page, lead, **opts)
    base = plain.run()
    for turn in range(3):
        e, f = ([(-60, 0, 45)[(s + turn) % 3] for s in range(3)], [(70, -50, 0)[(s + turn) % 3] for s in range(3)])
        times = lambda x, n: (x.double() * 2.0 ** n).to(torch.bfloat16)  # noqa: E731
        q2 = torch.cat([times(q[plain.of(s)], -e[s]) for s in range(3)])
        p = Pass(ops, seqs, [(times(k, e[s]), times(v, f[s])) for s, (k, v) in enumerate(kv)], q2, group, page, lead, **opts)
        got = p.run()
        for s in range(3):
            assert torch.equal(got[p.of(s)], times(base[p.of(s)], f[s])), (turn, s)


@pytest.mark.parametrize("by", [-11, -20, -40])
@pytest.mark.parametrize("what", ["k", "v", "group of v"])
@pytest.mark.parametrize("D,group,page", [(128, 32, 64), (64, 32, 16)])
def test_small_numbers_behind_a_window_keep_their_bits(ops, by, what, D, group, page):
    """Rows that see nothing but tokens far smaller than earlier ones of their sequence (or a group of them that is): as right as over a cache in bf16."""
    n, turn, window, Q, H = 700, 300, 130, 4, 2
    k, v = _kv([n], H, D, 3)[0]
    small = slice(turn, None), slice(None), slice(group if what == "group of v" else 0, None)
    x = k if what == "k" else v
    x[small] = (x[small].double() * 2.0 ** by).to(x.dtype)
    q = torch.randn(n, Q, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    if what == "k":
        q[turn + window:] = (q[turn + window:].double() * 2.0 ** -by).to(q.dtype)
    got = Pass(ops, [(0, n)], [(k, v)], q, group, page, window=window).run()[turn + window:]
    (kc, ks, kz), (vc, vs, vz) = quantised(k[turn:], group), quantised(v[turn:], group)
    kept = (values(kc, ks, kz, group), values(vc, vs, vz, group), ks, kz, vs)
    x, half = q[turn + window:], 2.0 ** -8
    want = attention(x, kept[0], kept[1], torch.arange(window, n - turn), scale=D ** -0.5, window=window)
    # (the floor for values of order one)
    tol = tolerance(x, kept, D ** -0.5, want, want[1], half, torch.bfloat16, group, value_step=half) - 1e-7
    assert ((got.double() - want[0]).abs() <= tol).all()
    # (sums that cancel take most of that: the outputs together are far closer)
    assert (got.double() - want[0]).norm() <= 2.0 ** -7 * want[0].norm()
    if what == "group of v":
        assert (got.double() - want[0])[..., group:].norm() <= 2.0 ** -7 * want[0][..., group:].norm()


@pytest.mark.parametrize("scale", [-0.11, 0.0, 0.07])
@pytest.mark.parametrize("opts", [{}, {"softcap": 3.0}, {"window": 50, "keep_first": 1}])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_portion_scales(ops, scale, opts, dt):
    """A factor of either sign, or zero, as for single tokens; queries and factor times powers of two that cancel change no bit."""
    seqs, Q, H, D, group = [(0, 300), (70, 3), (200, 129)], 4, 2, 128, 32
    kv = [(k.to(dt), v.to(dt)) for k, v in _kv([a + b for a, b in seqs], H, D, 7)]
    q = torch.randn(sum(b for _, b in seqs), Q, D, generator=torch.Generator().manual_seed(3)).to(dt)
    p = Pass(ops, seqs, kv, q, group, 64, sm_scale=scale, **opts)
    got = p.run()
    for s, (a, b) in enumerate(seqs):
        (kc, ks, kz), (vc, vs, vz) = (quantised(x, group) for x in kv[s])
        kept = (values(kc, ks, kz, group), values(vc, vs, vz, group), ks, kz, vs)
        x, half = q[p.of(s)], 2.0 ** -11
        want = attention(x, kept[0], kept[1], torch.arange(a, a + b), scale=scale, **opts)
        tol = tolerance(x, kept, abs(scale), want, want[1], half, dt, group, value_step=half)
        # (as in test_portions: below 2^-14 of the largest of the head, in steps of 2^-24)
        floor = 2.0 ** -24 * kept[0].abs().amax() * x.double().abs().sum(-1) * abs(scale)
        tol = tol + torch.expm1(2 * floor)[..., None] * want[1] + 2.0 ** -24 * kept[1].abs().amax()
        assert ((got[p.of(s)].double() - want[0]).abs() <= tol).all(), s
    # (fp16 has no more room for queries of order one)
    for e in (-100, -30, 30, 100) if dt is torch.bfloat16 else (-3, 5):
        q2 = (q.double() * 2.0 ** e).to(dt)
        keep = (q2.double() * 2.0 ** -e == q.double()).all(-1)
        again = Pass(ops, seqs, kv, q2, group, 64, sm_scale=scale * 2.0 ** -e, **opts).run()
        assert torch.equal(again[keep], got[keep]) and keep.float().mean() > 0.9, e


@pytest.mark.parametrize("opts", [{}, {"softcap": 3.0}, {"window": 50, "keep_first": 1}])
@pytest.mark.parametrize("e,f", [(-90, -90), (-60, -99), (-110, -110), (-95, 0)])
def test_scores_of_nothing(ops, opts, e, f):
    """Keys times 2^e and queries times 2^f: scores far below what fp32 tells from zero weigh all visible keys alike."""
    seqs, Q, H, D, group = [(0, 300), (70, 3), (200, 129)], 4, 2, 64, 32
    times = lambda x, n: (x.double() * 2.0 ** n).to(torch.bfloat16)  # noqa: E731
    kv = [(times(k, e), v) for k, v in _kv([a + b for a, b in seqs], H, D, 17)]
    q = times(torch.randn(sum(b for _, b in seqs), Q, D, generator=torch.Generator().manual_seed(3)), f)
    p = Pass(ops, seqs, kv, q, group, 64, **opts)
    got = p.run()
    for s, (a, b) in enumerate(seqs):
        vc, vs, vz = quantised(kv[s][1], group)
        v = values(vc, vs, vz, group)
        want = attention(q[p.of(s)], torch.zeros_like(v), v, torch.arange(a, a + b), scale=0.0, **opts)
        # values and weights in bf16 at the worst, and the output
        assert ((got[p.of(s)].double() - want[0]).abs() <= (2.0 ** -7 + 2.0 ** -15) * want[1] + 2.0 ** -8 * want[0].abs() + 2.0 ** -24 * v.abs().amax()).all(), s


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("opts", [{}, {"window": 100, "keep_first": 3, "sink": True}])
@pytest.mark.parametrize("lead", [0, 3])
def test_some_heads_at_a_time(ops, monkeypatch, dt, opts, lead):
    """Scratch of a fixed size, whatever the pages of a pass: outputs bit for bit those of one round, large numbers in some heads or not."""
    seqs, Q, H, D, group, page = [(900, 300), (0, 129), (77, 1)], 10, 5, 64, 32, 16
    kv = [(k.to(dt), v.to(dt)) for k, v in _kv([a + b for a, b in seqs], H, D, 21)]
    if dt is torch.bfloat16:
        kv[0][0][5, 3, 1] = 2.0 ** 40
    q = torch.randn(sum(b for _, b in seqs), Q, D, generator=torch.Generator().manual_seed(2)).to(dt)
    opts = dict(opts)
    if opts.pop("sink", False):
        opts["sink"] = torch.randn(Q, generator=torch.Generator().manual_seed(1)).to(dt)
    p = Pass(ops, seqs, kv, q, group, page, lead, **opts)
    want, same = p.run(), lambda a, b: torch.allclose(a, b, rtol=0, atol=0, equal_nan=True)  # (a score past 2^31 is no number)
    assert want.isfinite().float().mean() > 0.8
    pages, entries = p.table.numel(), 4
    whole, one = (ops._quant_portion(pages, lead, entries, h, D, page, ops._DT[dt], 1 << 40)[1] for h in (H, 1))
    for room in (whole - 1, whole // 2, 2 * one + 1, one, 1):
        monkeypatch.setattr(ops, "QUANT_PORTION_BYTES", room)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got = p.run()
        # (beside the scratch: tables, queries and output, and the allocator's 512 bytes of each)
        assert torch.cuda.max_memory_allocated() - before <= max(room, one) + 3 * q.numel() * 2 + 65536
        assert same(got, want), room
        ws = torch.empty(max(room, one) // 256 * 256 + 256, dtype=torch.uint8, device=DEV)
        p.opts["workspace"] = ws
        assert same(p.run(), want), room
        del p.opts["workspace"]
    for bad in (torch.empty(one - 1, dtype=torch.uint8, device=DEV), torch.empty(whole, dtype=torch.int8, device=DEV), torch.empty(whole + 8, dtype=torch.uint8, device=DEV)[8:],
                torch.empty(2 * whole, dtype=torch.uint8, device=DEV)[::2]):
        p.opts["workspace"] = bad
        with pytest.raises(ValueError, match="workspace"):
            p.run()


def test_an_engine_reserves_what_portions_take(ops, monkeypatch):
    """Long prompts, and portions beside them, take no memory that the engine has not had since it was made."""
    from blitz_scale_b200.runtime import core
    from blitz_scale_b200.runtime.engine import Engine
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 4096, (n,), generator=g).tolist() for n in (3000, 17, 900)]
    steps = [[2000, 0, 500], [500, 16, 399], [500, 1, 1]]
    outs = []
    for room in (1 << 28, 1 << 20):
        monkeypatch.setattr(ops, "QUANT_PORTION_BYTES", room)
        eng = Engine("tiny_gpu_wide", num_pages=256, page_size=16, max_batch=8, max_batch_tokens=4096, seed=0, kv_bits=4)
        reserved = eng.runner._ws["portion"]
        assert reserved.numel() <= max(room, 256 * 16 * 4 * 128 + 65536)
        b = eng.new_batch(1, [core.SeqSpec(i, p, 6) for i, p in enumerate(prompts)])
        got = []
        for counts in steps:
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            got.append(eng.step(b, counts, [[c - 1] if c else [] for c in counts]))
            assert torch.cuda.max_memory_allocated() - before <= 1 << 20        # (logits, tables)
        assert eng.runner._ws["portion"] is reserved
        outs.append(torch.cat(got))
    assert torch.equal(*outs)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("what", ["k", "v", "both"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_no_number_reaches_rows_that_see_it(ops, dt, shape, what, bad):
    """Rows before a token with such a key or value, rows whose window leaves it out, other heads and other sequences are bit for bit what they are without it."""
    seqs, Q, H, D, group, page, lead, opts = SHAPES[shape]
    kv = [(k.to(dt), v.to(dt)) for k, v in _kv([a + b for a, b in seqs], H, D, 50 * shape + 3)]
    q = torch.randn(sum(b for _, b in seqs), Q, D, generator=torch.Generator().manual_seed(shape)).to(dt)
    want = Pass(ops, seqs, kv, q, group, page, lead, **opts).run()
    first, n = seqs[1]
    at, rep = first + n // 2, Q // H
    k, v = (x.clone() for x in kv[1])
    if what != "v":
        k[at, 1, 3] = bad
    if what != "k":
        v[at, 1, D - 1] = bad
    p = Pass(ops, seqs, [kv[0], (k, v), kv[2]], q, group, page, lead, **opts)
    got = p.run()
    window = opts.get("window") or 1 << 30
    sees = torch.zeros(got.shape[:2], dtype=torch.bool)
    rows_at = torch.arange(first, first + n)
    sees[p.of(1), rep:2 * rep] = ((rows_at >= at) & (rows_at < at + window))[:, None]
    assert torch.equal(got[~sees], want[~sees])
    last = got[sees][:, D - group:]             # (the group that holds the value; a key reaches all)
    assert last.isnan().all() and sees.any()


@pytest.mark.parametrize("own_room", [False, True])
def test_captured_and_replayed(ops, own_room):
    """Two passes in a graph, one after the other in the same scratch, with other numbers at each replay: some held in fp16, some in bf16."""
    shapes, passes = [SHAPES[0], SHAPES[1]], []
    for i, (seqs, Q, H, D, group, page, lead, opts) in enumerate(shapes):
        kv = _kv([a + b for a, b in seqs], H, D, 90 + i)
        q = torch.randn(sum(b for _, b in seqs), Q, D, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16)
        passes.append((Pass(ops, seqs, kv, q, group, page, 0, **opts), kv))
    room = torch.empty(1 << 24, dtype=torch.uint8, device=DEV) if own_room else None
    calls = []
    for p, _ in passes:
        args = (p.q.flatten(1).to(DEV), p.cache, p.table.to(torch.int32).to(DEV), ops.prefill_work_list(p.rows, p.lens, p.page, DEV))
        more = dict(q_heads=p.q.shape[1], kv_heads=p.H, head_dim=p.D, page_size=p.page, workspace=room, **p.opts)
        calls.append(lambda out, args=args, more=more: ops.attn_prefill_paged(*args, out=out, **more))
    outs = [torch.zeros(p.q.shape[0], p.q.shape[1] * p.D, dtype=torch.bfloat16, device=DEV) for p, _ in passes]
    for call, out in zip(calls, outs):
        call(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call, out in zip(calls, outs):
            call(out)
    for by in (0, 25, 3, 40):
        for p, kv in passes:            # a key and a value of the first sequence grow
            k, v = (x[:1].clone() for x in kv[0])
            k[0, 0, 1], v[0, 0, 2] = 2.0 ** min(by, 20), -(2.0 ** by)
            slot = (p.table[:1] * p.page).to(torch.int32).to(DEV)
            ops.quant_kv_store(k.flatten(1).to(DEV), v.flatten(1).to(DEV), slot, p.cache)
        graph.replay()
        got = [o.clone() for o in outs]
        for call, out, g in zip(calls, outs, got):
            out.fill_(7.0)
            call(out)
            assert torch.equal(out, g) and g.isfinite().all(), by


@pytest.mark.parametrize("H,rep,D,group,page", [(130, 1, 64, 64, 16), (1, 40, 128, 128, 1024)])
def test_many_heads_and_large_pages(ops, H, rep, D, group, page):
    seqs = [(0, 37), (700, 5)]
    kv = _kv([a + b for a, b in seqs], H, D, 60)
    q = torch.randn(42, H * rep, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    p = Pass(ops, seqs, kv, q, group, page)
    got = p.run()
    for s, (a, b) in enumerate(seqs):
        kept = [quantised(x, group) for x in kv[s]]
        (kc, ks, kz), (vc, vs, vz) = kept
        kept = (values(kc, ks, kz, group), values(vc, vs, vz, group), ks, kz, vs)
        x, half = q[p.of(s)], 2.0 ** -11
        want = attention(x, kept[0], kept[1], torch.arange(a, a + b), scale=D ** -0.5)
        tol = tolerance(x, kept, D ** -0.5, want, want[1], half, torch.bfloat16, group, value_step=half)
        # (as in test_portions: below 2^-14 of the largest of the head, in steps of 2^-24)
        floor = 2.0 ** -24 * kept[0].abs().amax() * x.double().abs().sum(-1) * D ** -0.5
        tol = tol + torch.expm1(2 * floor)[..., None] * want[1] + 2.0 ** -24 * kept[1].abs().amax()
        assert ((got[p.of(s)].double() - want[0]).abs() <= tol).all(), s
