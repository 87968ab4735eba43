"""One workspace for decode attention over a 4-bit cache, and calls of different batch sizes with it."""
import itertools

import pytest
import torch

from test_quant_kv_gpu import DEV, rows

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


def _calls(ops, sizes, Q, H, D, group, page, seed=0):
    """(call(out, workspace), rows) of batches of so many sequences of so many tokens, whose pages are any of 64 filled ones."""
    g = torch.Generator().manual_seed(seed)
    pages = 64
    cache = ops.quant_kv_pool(pages, page, H, D, group)
    for p in range(0, pages, 16):
        k, v = (rows(16 * page, H, D, torch.bfloat16, seed + p + i).flatten(1).to(DEV) for i in range(2))
        ops.quant_kv_store(k, v, torch.arange(p * page, (p + 16) * page, dtype=torch.int32, device=DEV), cache)
    calls = []
    for n, tokens in sizes:
        each = -(-tokens // page)
        table = torch.randint(0, pages, (n * each,), generator=g).to(torch.int32).to(DEV)
        indptr = (torch.arange(n + 1) * each).to(torch.int32).to(DEV)
        last = torch.full((n,), (tokens - 1) % page + 1, dtype=torch.int32, device=DEV)
        q = torch.randn(n, Q * D, generator=g).to(torch.bfloat16).to(DEV)

        def call(out, ws, q=q, table=table, indptr=indptr, last=last):
            ops.attn_decode(q, cache, table, indptr, last, q_heads=Q, kv_heads=H, head_dim=D, page_size=page, num_splits=0, out=out, workspace=ws)
        calls.append((call, n))
    return calls


@pytest.mark.parametrize("Q,H,D,group,sizes", [
    (32, 8, 128, 32, [(2, 4000), (32, 800), (64, 2048), (128, 2048), (1, 4096), (256, 512)]),
    (8, 1, 64, 64, [(1, 30000), (70, 900), (3, 5000), (200, 300)]),
    (40, 8, 128, 128, [(1, 9000), (17, 1500), (120, 700), (2, 2500)]),
])
def test_batches_of_any_size_share_a_workspace(ops, Q, H, D, group, sizes):
    """A call's sums are never where another call has its tickets: outputs are bit for bit those of a workspace of the call's own, in whatever
    order the sizes come, and the tickets are zero after each."""
    calls = _calls(ops, sizes, Q, H, D, group, 64)
    want = []
    for call, n in calls:
        out = torch.full((n, Q * D), float("nan"), dtype=torch.bfloat16, device=DEV)
        call(out, torch.zeros(ops.quant_attn_workspace_bytes(n, Q, D), dtype=torch.uint8, device=DEV))
        assert out.isfinite().all()
        want.append(out)
    most, tickets = max(n for n, _ in sizes), ops.quant_attn_workspace_bytes(0, Q, D)
    ws = torch.zeros(ops.quant_attn_workspace_bytes(most, Q, D), dtype=torch.uint8, device=DEV)
    for order in itertools.islice(itertools.permutations(range(len(sizes))), 0, None, 17 if len(sizes) > 4 else 1):
        for i in order:
            out = torch.full_like(want[i], float("nan"))
            calls[i][0](out, ws)
            assert torch.equal(out, want[i]), (order, i)
            assert not ws[tickets:].any(), (order, i)


def test_heads_of_both_sizes_share_a_workspace(ops):
    """Where the tickets are does not depend on the size of the heads or on their number either."""
    a = _calls(ops, [(1, 9000), (90, 700)], 8, 2, 128, 32, 64)
    b = _calls(ops, [(1, 9000), (90, 700)], 16, 4, 64, 32, 64, seed=5)
    ws = torch.zeros(max(ops.quant_attn_workspace_bytes(90, 8, 128), ops.quant_attn_workspace_bytes(90, 16, 64)), dtype=torch.uint8, device=DEV)
    for one, two in ((a[0], b[1]), (b[0], a[1]), (a[0], a[1]), (b[0], b[1])):
        for call, n in (one, two):
            width = 8 * 128
            want, got = (torch.full((n, width), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
            call(want, None)
            call(got, ws)
            assert torch.equal(want, got) and want.isfinite().all()


@pytest.mark.parametrize("Q,H,D,group", [(32, 8, 128, 32), (8, 1, 64, 64)])
def test_a_call_that_gave_up_leaves_the_tickets_zero(ops, Q, H, D, group):
    """A wait that ran out is an error that the host reads, and the next call with this workspace is right."""
    sizes = [(2, 4000), (70, 900)]
    calls = _calls(ops, sizes, Q, H, D, group, 64)
    ws, tickets = torch.zeros(ops.quant_attn_workspace_bytes(70, Q, D), dtype=torch.uint8, device=DEV), ops.quant_attn_workspace_bytes(0, Q, D)
    want = [torch.empty(n, Q * D, dtype=torch.bfloat16, device=DEV) for n, _ in sizes]
    for (call, _), out in zip(calls, want):
        call(out, ws)
    for (call, _), out in zip(calls, want):
        got = torch.empty_like(out)
        ops.lib().blitz_attn_decode_quant_give_up(1)
        try:
            call(got, ws)
        finally:
            ops.lib().blitz_attn_decode_quant_give_up(0)
        with pytest.raises(RuntimeError, match="timed out"):
            ops.check_status()
        assert not ws[tickets:].any()
        call(got, ws)
        assert torch.equal(got, out)


@pytest.mark.parametrize("graphs", [False, True])
def test_an_engine_whose_batch_changes(ops, graphs):
    """Requests of a thousand tokens and more, batches of one to sixty of them in turn: the tokens of every step are those of a runner whose
    workspace is new."""
    from blitz_scale_b200.runtime import core
    from blitz_scale_b200.runtime.engine import Engine
    g = torch.Generator().manual_seed(1)
    lens = [1000 + 131 * (i % 9) for i in range(64)]
    lens[0], lens[20] = 6000, 5000
    prompts = [torch.randint(0, 4096, (n,), generator=g).tolist() for n in lens]
    runs = []
    for clean in (False, True):
        eng = Engine("tiny_gpu_wide", num_pages=2000, page_size=64, max_batch=64, max_batch_tokens=8192, seed=0, kv_bits=4, use_graphs=graphs)
        batches = []
        for i, (first, end) in enumerate(((0, 1), (1, 4), (4, 64))):
            for s in range(first, end, 3):          # (a pass of prompts holds 8192 tokens)
                part = eng.new_batch(100 * i + s, [core.SeqSpec(r, prompts[r], 12) for r in range(s, min(end, s + 3))])
                eng.prefill(part)
                if s > first:
                    batches[i].extend(part)
                else:
                    batches.append(part)
        steps = []
        for b in (0, 2, 1, 2, 0, 1, 0, 2):
            if clean and "quant" in eng.runner._ws:
                eng.runner._ws["quant"].zero_()
            steps.append((list(eng.decode(batches[b])), eng.runner.logits[:batches[b].size].clone()))
        runs.append(steps)
    for (a, x), (b, y) in zip(*runs):
        assert a == b and torch.equal(x, y)
