"""The largest numbers of a type in a 4-bit cache: a scale that is rounded up carries them past it, and nothing that reads the cache goes along."""
import pytest
import torch

from quant_kv_plain import attention, quantised, values
from test_quant_kv_gpu import DEV

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


@pytest.mark.parametrize("lens", [[1], [40], [9000, 3], [700] * 30])
@pytest.mark.parametrize("D,group", [(128, 32), (128, 128), (64, 64)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_single_tokens_over_the_largest_numbers_of_fp16(ops, lens, D, group, sign):
    """Values near 65504 whose last code stands for more: their weighted mean is a number, as it is where rows, pages and portions read them."""
    H, rep, page, dt = 2, 4, 64, torch.float16
    n = max(lens)
    # (from 0 to 65504: z = 0, s = 4384, and the last code stands for 65760; from -65504 to 0: z = -65536.  From 65520 on fp16 has infinity)
    v = torch.full((n, H, D), 65504.0) * sign
    v[:, :, ::group] = 0.0
    v = v.to(dt)
    k = torch.randn(n, H, D, generator=torch.Generator().manual_seed(1)).to(dt)
    table, used, slots = [], -(-n // page), torch.arange(n, dtype=torch.int32, device=DEV)
    cache = ops.quant_kv_pool(used, page, H, D, group)
    ops.quant_kv_store(k.flatten(1).to(DEV), v.flatten(1).to(DEV), slots, cache)
    vc, vs, vz = quantised(v, group)
    held = values(vc, vs, vz, group)
    assert held.abs().max() >= 65520
    indptr = [0]
    for m in lens:
        table += range(-(-m // page))
        indptr.append(len(table))
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    more = dict(q_heads=rep * H, kv_heads=H, head_dim=D, page_size=page)
    q = torch.randn(len(lens), rep * H * D, generator=torch.Generator().manual_seed(2)).to(dt)
    got = ops.attn_decode(q.to(DEV), cache, t(table), t(indptr), t([(m - 1) % page + 1 for m in lens]), **more).cpu().view(len(lens), -1, D)
    assert got.isfinite().all()
    for s, m in enumerate(lens[:3]):
        (kc, ks, kz) = quantised(k[:m], group)
        want = attention(q[s:s + 1].view(1, -1, D), values(kc, ks, kz, group), held[:m], torch.tensor([m - 1]), scale=D ** -0.5)[0]
        want = want.clamp(-65504.0, 65504.0)
        # (all tokens have the same values, so weights do not matter) weights times scales in fp16, their products with codes between -8 and 7, and sums, of
        # less than 65520 altogether; the rounding of the output
        assert ((got[s].double() - want[0]).abs() <= 65520 * (2.0 ** -11 + 2.0 ** -15 + m / 16 * 2.0 ** -22) + 2.0 ** -11 * want[0].abs()).all()
    # rows, pages and portions agree
    for y in (ops.quant_kv_load(cache, slots, dtype=dt)[1], ops.quant_kv_pages(cache, t(list(range(used))), dtype=dt)[:, 1].flatten(0, 1)[:n]):
        assert torch.equal(y.cpu(), held.clamp(-65504.0, 65504.0).to(dt))
    work = ops.prefill_work_list([1], [n], page, DEV)
    one = ops.attn_prefill_paged(q[:1].to(DEV), cache, t(list(range(used))), work, **more)
    assert one.isfinite().all()


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_single_tokens_over_the_largest_number_of_bf16(ops, sign):
    """One token, whose value is the largest number there is, beside zeros."""
    H, D, group, page, most = 2, 64, 32, 16, torch.finfo(torch.bfloat16).max
    v = torch.full((1, H * D), most * sign, dtype=torch.bfloat16)
    v[:, ::group] = 0.0
    cache, t = ops.quant_kv_pool(1, page, H, D, group), lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    ops.quant_kv_store(torch.ones_like(v).to(DEV), v.to(DEV), t([0]), cache)
    got = ops.attn_decode(torch.ones(1, 4 * H * D, dtype=torch.bfloat16, device=DEV), cache, t([0]), t([0, 1]), t([1]), q_heads=4 * H, kv_heads=H, head_dim=D,
                          page_size=page).cpu().view(H, 4, D)
    held = ops.quant_kv_load(cache, t([0]))[1].cpu().view(H, 1, D)
    assert held.isfinite().all() and got.isfinite().all()
    # (a row of one token is that token: rounded once, by weights of one)
    assert ((got.double() - held.double()).abs() <= 2.0 ** -7 * most).all()


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("n", [1, 50])
def test_portions_over_the_largest_number_of_bf16(ops, sign, n):
    """Rows whose own value has all of the weight: the largest number stays one."""
    H, D, group, page, most = 2, 64, 32, 64, torch.finfo(torch.bfloat16).max
    v = torch.full((n, H * D), most * sign, dtype=torch.bfloat16)
    v[:, ::group] = 0.0
    k = torch.zeros(n, H, D, dtype=torch.bfloat16)
    k[torch.arange(n), :, torch.arange(n)] = 64.0          # (keys at right angles, queries 64 times their own: every other weight is zero in fp32)
    cache, t = ops.quant_kv_pool(1, page, H, D, group), lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    ops.quant_kv_store(k.flatten(1).to(DEV), v.to(DEV), t(list(range(n))), cache)
    got = ops.attn_prefill_paged((64 * k).flatten(1).to(DEV), cache, t([0]), ops.prefill_work_list([n], [n], page, DEV), q_heads=H, kv_heads=H, head_dim=D,
                                 page_size=page).cpu()
    held = ops.quant_kv_load(cache, t(list(range(n))))[1].cpu().flatten(1)
    assert held.isfinite().all() and torch.equal(got, held)
