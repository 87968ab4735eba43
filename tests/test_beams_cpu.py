"""Beam search over a paged cache: what its calls refuse (on the CPU)."""
import pytest
import torch

from blitz_scale_b200 import ops

i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731


def _refused(call, *bad):
    for error, args, more in bad:
        with pytest.raises(error):
            call(*args, **more)


def test_select():
    z, s = torch.zeros(6, 50, dtype=torch.bfloat16), torch.zeros(6)
    _refused(ops.beam_select,
             (TypeError, (z.double(), s, 3), {}), (TypeError, (z.int(), s, 3), {}),
             (ValueError, (z[0], s, 3), {}), (ValueError, (z[:, :0], s, 3), {}), (ValueError, (z.t(), torch.zeros(50), 2), {}),
             (ValueError, (z, s, 4), {}), (ValueError, (z, s, 0), {}), (ValueError, (z, s, 65), {}),
             (ValueError, (z, s, 3), dict(n=65)), (ValueError, (z, s, 3), dict(n=-1)), (ValueError, (z, s, 3), dict(n=2, keep=3)), (ValueError, (z, s, 3), dict(keep=-1)),
             (ValueError, (z, s[:5], 3), {}), (ValueError, (z, s.double(), 3), {}), (ValueError, (z, torch.zeros(12)[::2], 3), {}),
             (ValueError, (z, s, 3), dict(ended=torch.zeros(2, dtype=torch.int64))), (ValueError, (z, s, 3), dict(ended=i32(2, 2))))
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.beam_select(z, s, 3)


def test_fork():
    table, cached, parents, pool = i32(6, 4), i32(6), i32(2, 3), i32(2, 9)
    more = dict(page_size=16, num_pages=20)
    _refused(ops.beam_fork,
             (ValueError, (table.long(), cached, parents, pool), more), (ValueError, (table[0], cached, parents, pool), more), (ValueError, (table[:5], cached, parents, pool), more),
             (ValueError, (table, cached[:5], parents, pool), more), (ValueError, (table, cached.long(), parents, pool), more), (ValueError, (table, i32(7), parents, pool), more),
             (ValueError, (table, cached, parents.long(), pool), more), (ValueError, (table, cached, parents.flatten(), pool), more),
             (ValueError, (table, cached, i32(2, 65), pool), more), (ValueError, (table, cached, i32(0, 3), pool), more), (ValueError, (table, cached, i32(3, 2).t(), pool), more),
             (ValueError, (table, cached, parents, pool.long()), more), (ValueError, (table, cached, parents, pool[:1]), more), (ValueError, (table, cached, parents, pool[0]), more),
             (ValueError, (table, cached, parents, pool), dict(more, page_size=0)), (ValueError, (table, cached, parents, pool), dict(more, num_pages=0)),
             (ValueError, (table, cached, parents, pool), dict(more, num_pages=1 << 21)), (ValueError, (table[:, :0], cached, parents, pool), more))
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.beam_fork(table, cached, parents, pool, **more)


def test_copies():
    cache, at = torch.zeros(5, 2, 16, 2, 64, dtype=torch.bfloat16), i32(3)
    _refused(ops.copy_pages,
             (ValueError, (cache, at.long(), at), {}), (ValueError, (cache, at, at[:2]), {}), (ValueError, (cache, at, at, at[:2]), {}), (ValueError, (cache, at.view(1, 3), at), {}),
             (ValueError, (cache, at, at, at.float()), {}), (ValueError, (cache, at, at), {}))


def test_tables():
    table, cached = i32(6, 4), i32(6)
    _refused(ops.step_tables,
             (ValueError, (table.long(), cached), dict(page_size=16)), (ValueError, (table[0], cached), dict(page_size=16)), (ValueError, (table, cached[:5]), dict(page_size=16)),
             (ValueError, (table, i32(7)), dict(page_size=16)), (ValueError, (table, cached.long()), dict(page_size=16)), (ValueError, (table, cached), dict(page_size=0)),
             (ValueError, (table, cached), dict(page_size=1 << 27)), (ValueError, (table, cached), dict(page_size=16, beams=4)), (ValueError, (table, cached), dict(page_size=16, beams=-1)),
             (ValueError, (table, cached), dict(page_size=16, tokens=9)), (ValueError, (table, cached), dict(page_size=16, entries=-1)),
             (ValueError, (table, cached, i32(5)), dict(page_size=16, tokens=9)), (ValueError, (table, cached, i32(6)), dict(page_size=16, tokens=-1)),
             (ValueError, (i32(8193, 1), i32(8193)), dict(page_size=16)), (ValueError, (table[:, :0], cached), dict(page_size=16)))
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.step_tables(table, cached, page_size=16)


def test_attention():
    q, kv = torch.zeros(4, 512, dtype=torch.bfloat16), torch.zeros(5, 2, 16, 2, 64, dtype=torch.bfloat16)
    args = (q, kv, i32(8), i32(5), i32(4), i32(2))
    more = dict(beams=2, q_heads=4, kv_heads=2, head_dim=64, page_size=16)

    def put(i, x):
        return args[:i] + (x,) + args[i + 1:]
    quant = ops.quant_kv_pool(4, 16, 2, 64, 32, device="cpu")
    pair = ops.KVPair(kv[:, 0].contiguous(), kv[:, 1].contiguous())
    _refused(ops.attn_decode_beams,
             (TypeError, put(0, q.float()), more), (ValueError, put(0, q[:3]), more), (ValueError, put(0, q[:, :255]), more), (ValueError, put(0, q[:, 1:]), more), (ValueError, put(0, q.t()), more),
             (ValueError, put(1, quant), more), (ValueError, put(1, pair), more), (ValueError, put(1, kv.half()), more), (ValueError, put(1, kv[:, :, :8]), more), (ValueError, put(1, kv[:0]), more),
             (ValueError, put(2, i32(8).long()), more), (ValueError, put(3, i32(6)), more), (ValueError, put(3, i32(4)), more), (ValueError, put(4, i32(3)), more),
             (ValueError, put(5, i32(1)), more), (ValueError, args, dict(more, beams=3)), (ValueError, args, dict(more, beams=0)), (ValueError, args, dict(more, q_heads=5)),
             (ValueError, args, dict(more, head_dim=32)), (ValueError, args, dict(more, page_size=24)), (ValueError, args, dict(more, page_size=8)), (ValueError, args, dict(more, kv_heads=0)),
             (ValueError, args, dict(more, softcap=-1.0)), (ValueError, args, dict(more, softcap=float("nan"))), (ValueError, args, dict(more, sink=torch.zeros(3, dtype=torch.bfloat16))),
             (ValueError, args, dict(more, sink=torch.zeros(4))), (ValueError, args, dict(more, out=torch.zeros(4, 256))), (ValueError, args, dict(more, out=torch.zeros(3, 256, dtype=torch.bfloat16))),
             (ValueError, args, dict(more, out=torch.zeros(4, 260, dtype=torch.bfloat16)[:, 1:257])))
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.attn_decode_beams(*args, **more)
