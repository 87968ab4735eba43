"""A cache held in 4 bits as an engine uses it: rotation with the write, whole steps, portions, graphs, sharing of workspaces."""
import math

import pytest
import torch

from quant_kv_plain import read_back

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def ops():
    from blitz_scale_b200 import ops as o
    o.lib()
    return o


@pytest.fixture(autouse=True)
def _status(ops):
    yield
    ops.check_status()


@pytest.mark.parametrize("T,Q,H,D,group,page,order", [(1, 4, 2, 128, 32, 64, "shuffled"), (7, 5, 1, 64, 64, 16, "shuffled"), (33, 32, 8, 128, 128, 64, "in order"),
                                                      (2500, 3, 2, 128, 64, 64, "in order"), (2401, 2, 1, 64, 32, 16, "in order"), (2400, 1, 3, 128, 32, 128, "shuffled")])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("static", [False, True])
def test_rotation_with_the_write(ops, T, Q, H, D, group, page, order, dt, static):
    """Queries and keys are rotated in place; the cache holds the quantised numbers of what the rows hold then."""
    g = torch.Generator().manual_seed(T)
    qkv = torch.randn(T, (Q + 2 * H) * D, generator=g).to(dt)
    pages = -(-T // page) + 2
    slot = torch.arange(page, page + T) if order == "in order" else torch.randperm(pages * page, generator=g)[:T]
    slot = slot.to(torch.int32)
    slot[T // 2] = -1                              # a row of padding
    pos = torch.randint(0, 16384, (T,), generator=g).to(torch.int32)
    cache = ops.quant_kv_pool(pages, page, H, D, group)
    dev = qkv.to(DEV)
    ops.rope_kv_store(dev, pos.to(DEV), slot.to(DEV), cache, q_heads=Q, kv_heads=H, head_dim=D, page_size=page, rope_theta=5e5, static_meta=static)
    got = dev.cpu()
    # an angle is off by half a step of fp32, of the frequency (2^-22 with the exponential) and of the product; the sum's rounding to fp32 and to the type
    x = qkv.double().view(T, Q + 2 * H, D)
    f = 5e5 ** (-torch.arange(0, D // 2).double() * 2 / D)
    a = pos.double()[:, None] * f
    c, s = a.cos()[:, None], a.sin()[:, None]
    lo, hi = x[:, :Q + H, :D // 2], x[:, :Q + H, D // 2:]
    want = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
    size = torch.cat([lo.abs() + hi.abs()] * 2, -1)
    off = torch.cat([a, a], -1)[:, None] * 2.0 ** -20 + 2.0 ** -20
    y = got.view(T, Q + 2 * H, D)
    assert ((y[:, :Q + H].double() - want).abs() <= HALF[dt] * want.abs() + off * size).all()
    assert torch.equal(y[:, Q + H:], qkv.view(T, Q + 2 * H, D)[:, Q + H:])
    k, v = ops.quant_kv_load(cache, slot.to(DEV), dtype=dt, k=torch.zeros(T, H, D, dtype=dt, device=DEV), v=torch.zeros(T, H, D, dtype=dt, device=DEV))
    keep = slot >= 0
    for h, z in ((k, y[:, Q:Q + H]), (v, y[:, Q + H:])):
        w = read_back(z, group)
        assert ((h.cpu().double() - w).abs() <= (HALF[dt] + 2.0 ** -23) * w.abs() + 2.0 ** -25)[keep].all()
        assert not h.cpu()[~keep].any()


def _engine(**more):
    from blitz_scale_b200.runtime.engine import Engine
    return Engine("tiny_gpu", num_pages=64, page_size=16, max_batch=8, max_batch_tokens=more.pop("tokens", 512), seed=0, **more)


def _batch(eng, prompts, new=6):
    from blitz_scale_b200.runtime import core
    b = eng.new_batch(1, [core.SeqSpec(i, p, new) for i, p in enumerate(prompts)])
    assert b is not None
    return b


def _prompts(lens):
    g = torch.Generator().manual_seed(5)
    return [torch.randint(0, 4096, (n,), generator=g).tolist() for n in lens]


class _Plain:
    """The model in fp32, whose attention reads the keys and values that the engine's cache holds of a sequence."""

    def __init__(self, eng):
        self.c = eng.cfg
        self.w = {n: eng.seg[n].float().cpu() for n in eng.seg.names()}

    def logits(self, tokens, cache):
        c, w = self.c, self.w
        norm = lambda x, g: x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + c.rms_eps) * g  # noqa: E731
        x, T, half = w["embed"][torch.tensor(tokens)], len(tokens), c.head_dim // 2
        a = torch.arange(T).float()[:, None] * c.rope_theta ** (-torch.arange(0, half).float() * 2 / c.head_dim)
        co, si = a.cos()[:, None], a.sin()[:, None]
        rot = lambda y: torch.cat([y[..., :half] * co - y[..., half:] * si, y[..., half:] * co + y[..., :half] * si], -1)  # noqa: E731
        own = []
        for l in range(c.layers):
            p = f"layers.{l}."
            qkv = (norm(x, w[p + "input_ln"]) @ w[p + "qkv"]).view(T, -1, c.head_dim)
            own.append((rot(qkv[:, c.q_heads:c.q_heads + c.kv_heads]), qkv[:, c.q_heads + c.kv_heads:]))
            q = rot(qkv[:, :c.q_heads])
            k, v = (y[:T].repeat_interleave(c.q_heads // c.kv_heads, 1) for y in cache[l])
            z = torch.einsum("thd,shd->hts", q, k) * c.head_dim ** -0.5
            z = z.masked_fill(torch.ones(T, T).triu(1).bool(), -math.inf)
            x = x + torch.einsum("hts,shd->thd", z.softmax(-1), v).reshape(T, -1) @ w[p + "o"]
            g, u = (norm(x, w[p + "post_ln"]) @ w[p + "gate_up"]).chunk(2, -1)
            x = x + (torch.nn.functional.silu(g) * u) @ w[p + "down"]
        return norm(x, w["final_norm"]) @ w["lm_head"], own


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("group", [32, 128])
def test_steps_of_an_engine_with_a_4_bit_cache(ops, graphs, group):
    """A portion of every prompt, then single tokens: logits are those of the plain model that reads the same cache, and the cache holds the
    model's own keys and values within half a step of their codes.  (A plain model that quantises its own keys would differ by codes next
    to a tie: activations that are off by 2^-9 turn about one in a hundred, by a whole step.)"""
    eng = _engine(kv_bits=4, kv_group=group, use_graphs=graphs)
    assert eng.kv.dtype == torch.uint8
    prompts = _prompts([5, 37, 100])
    b = _batch(eng, prompts)
    cuts = [[len(p) - 2 for p in prompts], [1] * 3, [1] * 3]
    got = [eng.step(b, c, [[n - 1] for n in c]).cpu() for c in cuts]
    plain, c = _Plain(eng), eng.cfg
    for r, p in enumerate(prompts):
        pages = torch.tensor(b.seqs[r].pages, dtype=torch.int32, device=DEV)
        cache = []
        for layer in eng.runner.kv:
            both = ops.quant_kv_pages(layer, pages, dtype=torch.float16).float().cpu()
            cache.append(tuple(both[:, i].reshape(-1, c.kv_heads, c.head_dim) for i in range(2)))
        for i, logits in enumerate(got):
            n = len(p) - 2 + i
            want, own = plain.logits(p[:n], cache)
            # (the bound that the 16-bit engine is held to: activations rounded to bf16 about ten times a layer)
            assert float((logits[r] - want[-1]).norm() / want[-1].norm()) < 2e-2
        for l in range(c.layers):
            for held, mine in zip(cache[l], own[l]):
                x = mine.unflatten(-1, (-1, group))
                step = (x.amax(-1) - x.amin(-1)) / 15 * (1 + 2.0 ** -7)
                # half a step, and 2e-2 of a row for activations that are not exactly these
                off = (held[:n].unflatten(-1, (-1, group)) - x).abs().amax(-1)
                assert (off <= step / 2 + 2e-2 * x.abs().amax()).all()


def test_decode_loop_graphs_and_layer_by_layer_agree(ops):
    prompts = _prompts([9, 64, 33, 17])
    outs = []
    for graphs in (False, True):
        eng = _engine(kv_bits=4, use_graphs=graphs)
        b = _batch(eng, prompts, new=12)
        toks = [eng.prefill(b)]
        for _ in range(8):
            toks.append(eng.decode(b))
        outs.append(toks)
    assert outs[0] == outs[1]


def test_portions_of_a_prompt_and_single_tokens_beside_them(ops):
    """A prompt in portions is the prompt in one pass (attention reads the same quantised keys either way): same cache bytes but for codes
    next to a tie, logits within rounding."""
    prompts = _prompts([300, 40])
    one, cut = _engine(kv_bits=4, tokens=512), _engine(kv_bits=4, tokens=512)
    a, b = _batch(one, prompts), _batch(cut, prompts)
    whole = one.step(a, [300, 40], [[299], [39]]).cpu()
    cut.step(b, [100, 0])
    cut.step(b, [120, 39])
    parts = cut.step(b, [80, 1], [[79], [0]]).cpu()
    assert float((whole - parts).norm() / whole.norm()) < 4e-2
    assert (one.kv != cut.kv).float().mean() < 0.05


def test_a_16_bit_engine_is_what_it_was(ops):
    eng = _engine()
    assert eng.kv.dtype == torch.bfloat16 and eng.kv_bits == 16 and not eng.runner.quant


def test_two_graphs_share_a_workspace_and_calls_on_another_stream(ops):
    """Tickets are zero after every call: graphs that share a workspace replay in any order, on whatever stream."""
    H, Q, D, group, page = 2, 8, 64, 32, 16
    g = torch.Generator().manual_seed(3)
    cache = ops.quant_kv_pool(40, page, H, D, group)
    k = torch.randn(600, H * D, generator=g).to(torch.bfloat16).to(DEV)
    ops.quant_kv_store(k, k.flip(0).contiguous(), torch.arange(600, dtype=torch.int32, device=DEV), cache)
    q = torch.randn(4, Q * D, generator=g).to(torch.bfloat16).to(DEV)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    index, more = torch.arange(40, dtype=torch.int32, device=DEV), dict(q_heads=Q, kv_heads=H, head_dim=D, page_size=page)
    tables = [(t([0, 10, 12, 12, 37]), t([3, 16, 0, 8])), (t([0, 37]), t([8]))]
    want = [ops.attn_decode(q[:p.numel() - 1], cache, index, p, last, **more) for p, last in tables]
    ws = torch.zeros(ops.quant_attn_workspace_bytes(4, Q, D), dtype=torch.uint8, device=DEV)
    outs, graphs = [torch.empty_like(w) for w in want], []
    torch.cuda.synchronize()
    for (p, last), o in zip(tables, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.attn_decode(q[:p.numel() - 1], cache, index, p, last, out=o, workspace=ws, **more)
        graphs.append(graph)
    side = torch.cuda.Stream()
    for order in ((0, 1), (1, 0, 0, 1)):
        for i in order:
            outs[i].fill_(7.0)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graphs[i].replay()
            torch.cuda.current_stream().wait_stream(side)
            assert torch.equal(outs[i], want[i])
    assert not ws[:256].any()
    assert torch.equal(want[0][2], torch.zeros_like(want[0][2]))


def test_many_sequences_and_a_long_one(ops):
    """More sequences than a launch's tables hold; one sequence over all blocks, whose pieces every block has some of."""
    H, Q, D, group, page = 1, 4, 64, 64, 16
    g = torch.Generator().manual_seed(4)
    cache = ops.quant_kv_pool(8, page, H, D, group)
    k = torch.randn(8 * page, D, generator=g).to(torch.bfloat16).to(DEV)
    ops.quant_kv_store(k, k, torch.arange(8 * page, dtype=torch.int32, device=DEV), cache)
    B = 1300
    lens = [(i * 7) % 40 for i in range(B)]
    indptr, index = [0], []
    for n in lens:
        index += [(n + j) % 8 for j in range(-(-n // page))]
        indptr.append(len(index))
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    q = torch.randn(B, Q * D, generator=g).to(torch.bfloat16).to(DEV)
    more = dict(q_heads=Q, kv_heads=H, head_dim=D, page_size=page)
    last = [(n - 1) % page + 1 if n else 0 for n in lens]
    out = ops.attn_decode(q, cache, t(index), t(indptr), t(last), **more)
    for i in (0, 1, 5, 40, 1023, 1024, 1025, 1299):
        alone = ops.attn_decode(q[i:i + 1], cache, t(index[indptr[i]:indptr[i + 1]] or [0]), t([0, indptr[i + 1] - indptr[i]]), t([last[i]]), **more)
        # (pieces are cut elsewhere: sums in another order, 2^-20 of weights' parts, rounded to bf16)
        assert (out[i] - alone[0]).float().abs().max() <= 2.0 ** -7 * max(1.0, float(alone.abs().max()))
    # the same eight pages over and over: the attention of 128 keys, whatever the length is a multiple of them
    many = 4000
    long = ops.attn_decode(q[:1], cache, t(list(range(8)) * many), t([0, 8 * many]), t([page]), **more)
    short = ops.attn_decode(q[:1], cache, t(list(range(8))), t([0, 8]), t([page]), **more)
    assert (long - short).float().abs().max() <= 2.0 ** -7 * max(1.0, float(short.abs().max()))


def test_what_is_no_number_reaches_those_that_see_it(ops):
    H, Q, D, group, page = 1, 2, 64, 32, 16
    g = torch.Generator().manual_seed(6)
    k, v = (torch.randn(70, D, generator=g).to(torch.bfloat16) for _ in range(2))
    v[20, 3] = math.nan                       # the first group of one value
    k[50, 40] = math.inf
    cache = ops.quant_kv_pool(5, page, H, D, group)
    ops.quant_kv_store(k.to(DEV), v.to(DEV), torch.arange(70, dtype=torch.int32, device=DEV), cache)
    q = torch.randn(1, Q * D, generator=g).to(torch.bfloat16).to(DEV)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    run = lambda n, **m: ops.attn_decode(q, cache, torch.arange(5, dtype=torch.int32, device=DEV), t([0, -(-n // page)]), t([(n - 1) % page + 1]),  # noqa: E731
                                         q_heads=Q, kv_heads=H, head_dim=D, page_size=page, **m).view(Q, D)
    assert run(20).isfinite().all()                                     # behind the end
    bad = run(21)
    assert bad[:, :32].isnan().all() and bad[:, 32:].isfinite().all()   # its group alone
    assert run(70).isnan().all()                                        # a key: every weight
    assert run(70, window=19).isfinite().all()                          # outside the window
    assert run(45, window=24).isfinite().all() and run(45, window=25)[:, :32].isnan().all()
    assert run(70, window=10, keep_first=5).isfinite().all()
