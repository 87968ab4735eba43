"""Attention of single tokens over a 4-bit cache whose values are of very different sizes: what has no weight costs nothing."""
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


def _run(ops, lens, k, v, q, group, page=64, **opts):
    """Sequences of so many tokens of k and v [n, heads, dim]."""
    n, H, D = k.shape
    used = -(-n // page)
    cache, t = ops.quant_kv_pool(used, page, H, D, group), lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    ops.quant_kv_store(k.flatten(1).to(DEV), v.flatten(1).to(DEV), torch.arange(n, dtype=torch.int32, device=DEV), cache)
    table, indptr = [], [0]
    for m in lens:
        table += range(-(-m // page))
        indptr.append(len(table))
    out = ops.attn_decode(q.flatten(1).to(DEV), cache, t(table), t(indptr), t([(m - 1) % page + 1 for m in lens]), q_heads=q.shape[1], kv_heads=H, head_dim=D,
                          page_size=page, **opts)
    return out.cpu().view(len(lens), -1, D)


def _kept(k, v, group):
    (kc, ks, kz), (vc, vs, vz) = quantised(k, group), quantised(v, group)
    return values(kc, ks, kz, group), values(vc, vs, vz, group), ks, kz, vs


STEP = 2.0 ** -11 + 2.0 ** -15          # of a weight times its scale, as for single tokens in general


@pytest.mark.parametrize("lens,places", [([700], (3,)), ([700, 40, 333], (0, 39)), ([20000, 300], (5, 250, 9000)), ([900] * 40, (450, 899)), ([1000, 200], tuple(range(70, 180))),
                                         ([6000], tuple(range(4000)))])
@pytest.mark.parametrize("rep,D,group", [(4, 128, 32), (8, 128, 32), (4, 64, 64), (1, 128, 64)])
@pytest.mark.parametrize("by", [25, 60, 100])
def test_large_values_without_weight(ops, lens, places, rep, D, group, by):
    """Tokens whose values are 2^by times the others' and whose scores are far below them for some heads, above for none: heads that give them no weight
    have outputs as right as without them."""
    n, H = max(lens), 2
    k, v = (rows(n, H, D, torch.bfloat16, 3 + i) for i in range(2))
    q = torch.randn(len(lens), rep * H, D, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    q[:, :, 0] = 16.0
    for p in places:
        k[p, :, 0], v[p] = -400.0, (v[p].double() * 2.0 ** by).to(torch.bfloat16)      # (scores of -16 * 400 / sqrt(D): no weight in fp32)
    got = _run(ops, lens, k, v, q, group)
    rest = torch.ones(n, dtype=torch.bool)
    rest[list(places)] = False
    for s, m in enumerate(lens[:3]):
        seen = rest[:m]
        kept = _kept(k[:m][seen], v[:m][seen], group)
        want = attention(q[s:s + 1], kept[0], kept[1], torch.tensor([int(seen.sum()) - 1]), scale=D ** -0.5)
        spread = attention(q[s:s + 1], kept[0], 8 * kept[4].repeat_interleave(group, -1), torch.tensor([int(seen.sum()) - 1]), scale=D ** -0.5)[0]
        tol = tolerance(q[s:s + 1], kept, D ** -0.5, want, spread, STEP + m / 16 * 2.0 ** -22, torch.bfloat16, group) + m * 2.0 ** -28 * kept[4].max()
        assert ((got[s].double() - want[0][0]).abs() <= tol[0]).all(), s
        assert (got[s].double() - want[0][0]).norm() <= 2.0 ** -7 * want[0][0].norm()


@pytest.mark.parametrize("rep,group", [(2, 32), (4, 32), (8, 64), (6, 128)])
@pytest.mark.parametrize("by", [20, 40])
@pytest.mark.parametrize("n", [200, 5000])
def test_large_values_that_some_heads_weigh(ops, rep, group, by, n):
    """Every other head gives a token with large values all of its weight, the others none of it."""
    H, D, place = 1, 128, 100
    k, v = (rows(n, H, D, torch.bfloat16, 13 + i) for i in range(2))
    q = torch.randn(1, rep, D, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    q[:, ::2, 0], q[:, 1::2, 0] = 16.0, -16.0
    k[:, :, 0] = 0.0
    k[place, :, 0], v[place] = 400.0, (v[place].double() * 2.0 ** by).to(torch.bfloat16)
    got = _run(ops, [n], k, v, q, group)[0].double()
    kept = _kept(k, v, group)
    want = attention(q, kept[0], kept[1], torch.tensor([n - 1]), scale=D ** -0.5)[0][0]
    for h in range(rep):
        assert (got[h] - want[h]).norm() <= 2.0 ** -7 * want[h].norm(), h


@pytest.mark.parametrize("rep,D,group", [(4, 128, 32), (8, 128, 64), (3, 64, 32)])
@pytest.mark.parametrize("order", [1, -1])
@pytest.mark.parametrize("n", [64, 300, 12000, 200000])
def test_scores_that_grow_and_values_that_fall(ops, rep, D, group, order, n):
    """Weights that rise by 2^100 and more along a sequence (or fall) while values fall by 2^40 (or rise), head by head as right as in 64 bits."""
    H, dt = 2, torch.bfloat16
    k, v = (rows(n, H, D, dt, 23 + i) for i in range(2))
    q = torch.randn(1, rep * H, D, generator=torch.Generator().manual_seed(7)).to(dt)
    q[:, :, 0] = 8.0
    at = (torch.arange(n) if order > 0 else torch.arange(n).flip(0)).double() / n
    k[:, :, 0] = (at * 200.0)[:, None].to(dt)
    v = (v.double() * torch.exp2(-(at * 40).floor())[:, None, None]).to(dt)
    got = _run(ops, [n], k, v, q, group)[0].double()
    kept = _kept(k, v, group)
    want = attention(q, kept[0], kept[1], torch.tensor([n - 1]), scale=D ** -0.5)
    for h in range(rep * H):
        assert (got[h] - want[0][0, h]).norm() <= 2.0 ** -6 * want[1][0, h].norm(), h


@pytest.mark.parametrize("rep,D,group", [(4, 128, 32), (8, 128, 32), (8, 64, 32)])
@pytest.mark.parametrize("by", [-10, -16, -20])
def test_groups_of_different_size(ops, rep, D, group, by):
    """A group of a head's values 2^by times as large as the others in every token."""
    n, H = 1500, 2
    k, v = (rows(n, H, D, torch.bfloat16, 33 + i) for i in range(2))
    v[:, :, group:2 * group] = (v[:, :, group:2 * group].double() * 2.0 ** by).to(torch.bfloat16)
    q = torch.randn(1, rep * H, D, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16)
    got = _run(ops, [n], k, v, q, group)[0].double()
    kept = _kept(k, v, group)
    want = attention(q, kept[0], kept[1], torch.tensor([n - 1]), scale=D ** -0.5)
    spread = attention(q, kept[0], 8 * kept[4].repeat_interleave(group, -1), torch.tensor([n - 1]), scale=D ** -0.5)[0]
    # (beside the largest scale at 2^6, what is below 2^-14 in steps of 2^-24, times codes up to 8)
    tol = tolerance(q, kept, D ** -0.5, want, spread, STEP + n / 16 * 2.0 ** -22, torch.bfloat16, group) - 1e-7 + n * 2.0 ** -28 * kept[4].max()
    assert ((got - want[0][0]).abs() <= tol[0]).all()
    small = got.view(rep * H, -1, group)[:, 1] - want[0][0].view(rep * H, -1, group)[:, 1]
    assert small.norm() <= 2.0 ** -7 * want[0][0].view(rep * H, -1, group)[:, 1].norm()


@pytest.mark.parametrize("rise", [0.65, 2.0, 11.0])
def test_weights_that_pass_bit_by_bit(ops, rise):
    """A token of large values is left behind by scores that rise a little from chunk to chunk: in the end it has no weight, and costs nothing."""
    H, rep, D, group, n = 1, 4, 128, 32, 6000         # (few heads: a warp has several chunks of a sequence, one after another)
    k, v = (rows(n, H, D, torch.bfloat16, 43 + i) for i in range(2))
    q = torch.randn(1, rep * H, D, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    q[:, :, 0] = 16.0
    k[:, :, 0] = (torch.arange(n) // 32 * rise).clamp(max=2000.0)[:, None].to(torch.bfloat16)
    for by in (0, 30, 80):
        big = v.clone()
        big[:8] = (v[:8].double() * 2.0 ** by).to(torch.bfloat16)
        for m in (64, 640, n):
            got = _run(ops, [m] * 150, k[:m], big[:m], q.expand(150, -1, -1).contiguous(), group)[0].double()
            kept = _kept(k[:m], big[:m], group)
            want = attention(q, kept[0], kept[1], torch.tensor([m - 1]), scale=D ** -0.5)
            for h in range(rep * H):
                assert (got[h] - want[0][0, h]).norm() <= 2.0 ** -6 * want[1][0, h].norm(), (by, m, h)
