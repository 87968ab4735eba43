"""Attention of beams where scores or values leave the ordinary range."""
import math

import pytest
import torch

import beams_plain as plain
from blitz_scale_b200 import ops

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731


def _case(common, tails, page, kvh, rep, dim, dtype, seed=0):
    """One request: `common` full pages of all beams, behind them tails[b] tokens of beam b's own."""
    g = torch.Generator("cuda").manual_seed(seed)
    lists, lengths, num = [], [], common
    for t in tails:
        lists.append([*range(common), *range(num, num - -t // page)])
        num -= -t // page
        lengths.append(common * page + t)
    kv = torch.randn(num + 1, 2, page, kvh, dim, generator=g, device="cuda").to(dtype)
    q = torch.randn(len(tails), kvh * rep * dim, generator=g, device="cuda").to(dtype)
    return q, kv, lists, lengths


def _run(q, kv, lists, lengths, common, kvh, rep, **more):
    indptr = [0]
    for x in lists:
        indptr.append(indptr[-1] + len(x))
    page, dim = kv.shape[2], kv.shape[4]
    out = ops.attn_decode_beams(q, kv, i32(sum(lists, [])), i32(indptr), i32([(n - 1) % page + 1 for n in lengths]), i32([common]), beams=len(lists), q_heads=kvh * rep,
                                kv_heads=kvh, head_dim=dim, page_size=page, **more)
    ops.check_status()
    return out


def _checked(q, kv, lists, lengths, common, kvh, rep, **more):
    """Against 64 bits: half a step of the type for the weights, as operands, times the largest value's size, half a step for the output (a quarter of that again for what
    scores of fp32 are off by)."""
    out = _run(q, kv, lists, lengths, common, kvh, rep, **more)
    want = plain.attend(q, kv, lists, lengths, kvh * rep, kvh, kv.shape[4], scale=more.get("sm_scale"), cap=more.get("softcap", 0.0), sink=more.get("sink"))
    half, top = torch.finfo(q.dtype).eps / 2, kv[:, 1].double().abs().max().item()
    assert torch.equal(out.isnan().cpu(), want.isnan())
    there = ~want.isnan()
    off = (out.double().cpu() - want).abs()[there]
    assert (off <= half * (want.abs()[there] + top * 1.25)).all(), (off.max().item(), half * top)


@pytest.mark.parametrize("page,kvh,rep,dim,dtype", [(64, 2, 4, 128, BF), (16, 2, 5, 64, BF), (64, 1, 8, 128, HF)])
@pytest.mark.parametrize("where", ["first tokens", "a page", "all that is common", "every second step", "all but the last token"])
def test_scores_of_minus_infinity(where, page, kvh, rep, dim, dtype):
    """Keys of minus infinity under positive queries: those tokens have no weight, and the others keep theirs."""
    common, tails = 3, [page + 20, 17, 2 * page, 1]
    q, kv, lists, lengths = _case(common, tails, page, kvh, rep, dim, dtype)
    q.abs_().add_(0.01)
    if where == "first tokens":
        for x in lists:
            for p in {x[0], x[common]}:
                kv[p, 0, :min(16, page - 1)] = -math.inf
    elif where == "a page":
        kv[1, 0] = -math.inf
    elif where == "all that is common":
        kv[:common, 0] = -math.inf
    elif where == "every second step":
        steps = kv.view(kv.shape[0], 2, page // 16, 16, kvh, dim)
        steps[:, 0].masked_fill_((torch.arange(kv.shape[0] * (page // 16), device="cuda") % 2 == 0).view(-1, page // 16, 1, 1, 1), -math.inf)
        for b, (x, n) in enumerate(zip(lists, lengths)):      # (every row has one token left at least)
            kv[x[(n - 1) // page], 0, (n - 1) % page] = 0.125 * (b + 1)
    else:
        for x, n in zip(lists, lengths):
            for p in x:
                kv[p, 0] = -math.inf
        for x, n in zip(lists, lengths):
            kv[x[(n - 1) // page], 0, (n - 1) % page] = 0.5
    for more in (dict(), dict(sm_scale=2.0), dict(sink=torch.linspace(-2.0, 2.0, kvh * rep, device="cuda").to(dtype))):
        _checked(q, kv, lists, lengths, common, kvh, rep, **more)


def test_rows_of_minus_infinity_alone():
    """Nothing has weight: no number, as a softmax of them; with a sink, which takes all of it, zeros."""
    q, kv, lists, lengths = _case(2, [5, 20, 1], 16, 2, 4, 64, BF)
    q.abs_().add_(0.01)
    kv[:, 0] = -math.inf
    _checked(q, kv, lists, lengths, 2, 2, 4)
    out = _run(q, kv, lists, lengths, 2, 2, 4, sink=torch.zeros(8, dtype=BF, device="cuda"))
    assert (out == 0).all()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_scores_of_the_largest_numbers(dtype):
    """Scores up to what fp32 holds: below the largest ones nothing has weight."""
    q, kv, lists, lengths = _case(3, [30, 5], 16, 1, 2, 64, dtype)
    q.fill_(1.0)
    big = torch.finfo(dtype).max / 128
    for p in range(kv.shape[0]):
        kv[p, 0] = -big
    kv[1, 0, 3], kv[1, 0, 9] = -big / 2, -big / 2
    for scale in (None, 1.0, 1.5):
        _checked(q, kv, lists, lengths, 3, 1, 2, **({} if scale is None else dict(sm_scale=scale)))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("common", [0, 8])
def test_values_near_the_largest_number(dim, common):
    """Values whose mean fp32 holds, behind scores that rise by 2^7.9 from step to step of a piece: weights are one at most, so that sums stay below tokens x values."""
    page, kvh, rep = 16, 1, 4
    q, kv, lists, lengths = _case(common, [64, 33], page, kvh, rep, dim, BF)
    q.fill_(1.0)
    kv[:, 0] = 0.0
    kv[1::2, 0, :, :, 0] = 7.875
    kv[:, 1] = kv[:, 1].abs().clamp(0.5, 1.0) * 1.5e36
    _checked(q, kv, lists, lengths, common, kvh, rep, sm_scale=math.log(2.0))


def test_calls_repeat_themselves():
    """The same call gives the same bits, whatever the warps' order was."""
    q, kv, lists, lengths = _case(70, [100, 37, 200, 1, 64, 9, 18, 77], 64, 8, 4, 128, BF)
    first = _run(q, kv, lists, lengths, 70, 8, 4)
    for _ in range(30):
        assert torch.equal(_run(q, kv, lists, lengths, 70, 8, 4), first)
