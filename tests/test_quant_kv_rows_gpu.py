"""Rows without a slot, read back from a 4-bit cache."""
import pytest
import torch

from test_quant_kv_gpu import DEV, SIZES, rows, stored

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


@pytest.mark.parametrize("D,group", SIZES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1, 7, 33, 200])
def test_rows_without_a_slot(ops, D, group, dt, T):
    """Zeros in outputs that the call makes, left as they are in those that it is given, in any mixture of both."""
    H, page = 3, 16
    k, v = rows(T, H, D, dt, 1), rows(T, H, D, dt, 2)
    slot = torch.randperm(256, generator=torch.Generator().manual_seed(T))[:T]
    cache = stored(ops, k, v, slot, H, D, group, page, 16)
    full = [x.cpu() for x in ops.quant_kv_load(cache, slot.to(torch.int32).to(DEV), dtype=dt)]
    none = torch.rand(T, generator=torch.Generator().manual_seed(T + 1)) < 0.4
    none[T // 2] = True
    some = torch.where(none, -1 - slot, slot).to(torch.int32).to(DEV)
    for given in ((), ("k",), ("v",), ("k", "v")):
        junk = torch.full((64 << 10,), 3.0, dtype=dt, device=DEV)         # (what new memory may hold)
        del junk
        out = {n: torch.full((T, H, D), 5.0, dtype=dt, device=DEV) for n in given}
        got = ops.quant_kv_load(cache, some, **(out or {"dtype": dt}))
        for n, y, want in zip("kv", got, full):
            y = y.cpu()
            assert torch.equal(y[~none], want[~none])
            assert (y[none] == (5.0 if n in given else 0.0)).all()
