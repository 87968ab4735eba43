"""A cache held in 4 bits: what its calls refuse (on the CPU), and the plain form's own arithmetic."""
import pytest
import torch

from blitz_scale_b200 import ops
from quant_kv_plain import down, quantised, read_back


def test_plain_numbers():
    a = torch.tensor([1.0, 1.0 + 2.0 ** -8, -1.0 - 2.0 ** -8, 0.0, 257.0, -3.0])
    assert torch.equal(down(a.double()), torch.tensor([1.0, 1.0, -1.0 - 2.0 ** -7, 0.0, 256.0, -3.0]).double())
    x = torch.randn(50, 64, generator=torch.Generator().manual_seed(0)).to(torch.float16)
    for group in (32, 64):
        c, s, z = quantised(x, group)
        assert c.min() == 0 and c.max() == 15
        assert ((read_back(x, group) - x.double()).abs() <= (s / 2).repeat_interleave(group, -1) * (1 + 1e-9)).all()
        y = x.double().unflatten(-1, (-1, group))
        assert (z <= y.amin(-1)).all() and (z + 15 * s >= y.amax(-1)).all()


@pytest.mark.parametrize("dim,group", [(96, 32), (128, 16), (64, 128), (256, 64), (128, 96)])
def test_sizes_refused(dim, group):
    with pytest.raises(ValueError):
        ops.quant_kv_block_bytes(dim, group)


@pytest.mark.parametrize("page", [8, 24, 0, 48])
def test_pages_refused(page):
    with pytest.raises(ValueError):
        ops.quant_kv_pool(2, page, 2, 64, 32, device="cpu")


def _pool(**more):
    return ops.quant_kv_pool(4, 16, 2, 64, 32, device="cpu")._replace(**more)


def test_caches_and_rows_refused():
    k, slot = torch.zeros(3, 128, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    good = _pool()
    for cache in (_pool(dim=128), _pool(group=64), good._replace(pool=good.pool.float()), good._replace(pool=good.pool[:, :1]),
                  good._replace(pool=good.pool[:, :, :, :-16])):
        with pytest.raises(ValueError):
            ops.quant_kv_store(k, k, slot, cache)
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.quant_kv_store(k, k, slot, good)
    for bad in (k.float(), k.double()):
        with pytest.raises(TypeError):
            ops._quant_rows(bad, 2, 64, "k")
    for bad in (k[:, :64], k.t(), k[:, 1:], torch.zeros(3, 132, dtype=torch.bfloat16)[:, :128], k.view(3, 4, 32), k.flatten()):
        with pytest.raises(ValueError):
            ops._quant_rows(bad, 2, 64, "k")
    for bad, n in ((slot.long(), 3), (slot, 4), (slot[::2], 1), (slot.view(1, 3), 3)):
        with pytest.raises(ValueError):
            ops._int32(bad, n, "slot")


def test_reading_back_refused():
    good, slot = _pool(), torch.zeros(3, dtype=torch.int32)
    for more in (dict(k=torch.zeros(3, 2, 32, dtype=torch.bfloat16)), dict(v=torch.zeros(3, 2, 64, dtype=torch.float16)),
                 dict(k=torch.zeros(2, 2, 64, dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            ops.quant_kv_load(good, slot, **more)
    with pytest.raises(ValueError):
        ops.quant_kv_pages(good, slot, out=torch.zeros(3, 2, 16, 2, 32, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        ops.quant_kv_pages(good, slot.long())


def test_attention_refused():
    good = _pool()
    q, t = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(8, dtype=torch.int32)
    base = dict(q_heads=4, kv_heads=2, head_dim=64, page_size=16)
    call = lambda q=q, indptr=t[:3], **more: ops.attn_decode(q, good, t, indptr, t[:2], **{**base, **more})  # noqa: E731
    for more in (dict(gate=q), dict(bias=q), dict(chunked=True), dict(sigmoid=True), dict(kv_heads=4), dict(head_dim=128), dict(page_size=32),
                 dict(q_heads=5), dict(q_heads=8), dict(window=-1), dict(keep_first=-1), dict(softcap=-1.0), dict(softcap=float("nan")),
                 dict(sink=torch.zeros(4)), dict(sink=torch.zeros(3, dtype=torch.bfloat16)), dict(num_splits=-1),
                 dict(out=torch.zeros(2, 128, dtype=torch.bfloat16)), dict(out=torch.zeros(2, 256)), dict(out=torch.zeros(1, 256, dtype=torch.bfloat16)),
                 dict(indptr=t[:4]), dict(indptr=t[:3].long()), dict(q=q[:, 1:]), dict(q=q.t())):
        with pytest.raises(ValueError):
            call(**more)
    with pytest.raises(TypeError):
        call(q=q.float())
    with pytest.raises(ValueError, match="current CUDA device"):
        call()
    work = torch.zeros(1, 8, dtype=torch.int32)
    for more in (dict(skip_pages=9), dict(skip_pages=-1), dict(gate=q), dict(work=work.long()), dict(work=work[0]), dict(out=torch.zeros(1, 256, dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            ops.attn_prefill_paged(q, good, t, **{**base, "work": work, **more})
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.attn_prefill_paged(q, good, t, work, **base)


def test_rotation_refused():
    good, qkv, t = _pool(), torch.zeros(3, 8 * 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    base = dict(q_heads=4, kv_heads=2, head_dim=64, page_size=16, rope_theta=1e4)
    for more in (dict(kv_heads=1), dict(head_dim=128), dict(page_size=64), dict(q_heads=3), dict(rope_theta=0.0), dict(rope_theta=float("nan"))):
        with pytest.raises(ValueError):
            ops.rope_kv_store(qkv, t, t, good, **{**base, **more})
    for bad in (qkv.t(), qkv[:, ::2], torch.zeros(6, 512, dtype=torch.bfloat16)[::2]):
        with pytest.raises(ValueError):
            ops.rope_kv_store(bad, t, t, good, **base)
    with pytest.raises(TypeError):
        ops.rope_kv_store(qkv.float(), t, t, good, **base)
    for pos, slot in ((t[:2], t), (t, t[:2]), (t.long(), t)):
        with pytest.raises(ValueError):
            ops.rope_kv_store(qkv, pos, slot, good, **base)
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.rope_kv_store(qkv, t, t, good, **base)


def test_bytes_of_a_page():
    from blitz_scale_b200.models.config import get_config
    from blitz_scale_b200.runtime.engine import kv_page_bytes
    c = get_config("llama3_8b")
    assert kv_page_bytes(c, 64) == 2 * 64 * 8 * 128 * 2 and kv_page_bytes(c, 64, tp=2) == 64 * 8 * 128 * 2
    # a token of a head: 64 bytes of codes and four pairs of 16-bit numbers, of its key and of its value
    assert kv_page_bytes(c, 64, kv_bits=4, kv_group=32) == 64 * 8 * 2 * (64 + 16)
    assert kv_page_bytes(c, 16, kv_bits=4, kv_group=128) == 16 * 8 * 2 * (64 + 4)
    pool = ops.quant_kv_pool(3, 64, 8, 128, 64, device="cpu")
    assert pool.pool[0].numel() == kv_page_bytes(c, 64, kv_bits=4, kv_group=64) and pool.kv_heads == 8 and pool.page_size == 64
    for more in (dict(kv_bits=8), dict(kv_bits=4, kv_group=16), dict(kv_bits=4, page_size=8)):
        with pytest.raises(ValueError):
            kv_page_bytes(c, more.pop("page_size", 64), **more)


def test_engines_that_take_no_4_bit_cache():
    from blitz_scale_b200.runtime.engine import Engine
    cpu = torch.device("cpu")
    with pytest.raises(ValueError, match="16 or 4 bits"):
        Engine("tiny", num_pages=4, device=cpu, kv_bits=8)
    for model, more in (("fafudra_tiny", {}), ("tiny", dict(tp=2))):
        with pytest.raises(ValueError, match="uniform models on one GPU"):
            Engine(model, num_pages=4, device=cpu, kv_bits=4, **more)


def test_caches_without_pages_refused():
    t, k = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 128, dtype=torch.bfloat16)
    empty = ops.quant_kv_pool(0, 16, 2, 64, 32, device="cpu")
    q, base = torch.zeros(2, 256, dtype=torch.bfloat16), dict(q_heads=4, kv_heads=2, head_dim=64, page_size=16)
    for call in (lambda: ops.quant_kv_store(k, k, t, empty), lambda: ops.quant_kv_load(empty, t), lambda: ops.quant_kv_pages(empty, t),
                 lambda: ops.attn_decode(q, empty, t, t, t[:2], **base), lambda: ops.attn_prefill_paged(q, empty, t, torch.zeros(1, 8, dtype=torch.int32), **base),
                 lambda: ops.rope_kv_store(torch.zeros(3, 8 * 64, dtype=torch.bfloat16), t, t, empty, rope_theta=1e4, **base)):
        with pytest.raises(ValueError, match="without pages"):
            call()
