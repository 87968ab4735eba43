"""Scratch of attention over a 4-bit cache: its sizes, and what is refused (on the CPU)."""
import pytest
import torch

from blitz_scale_b200 import ops


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,dim,page", [(8, 128, 64), (1, 64, 16), (5, 128, 128), (32, 64, 16)])
def test_a_pass_of_fewer_pages_fits_where_more_do(dtype, heads, dim, page):
    dt, entries = ops._DT[dtype], 300
    for pages in (1, 7, 130, 2048, 30000):
        room = ops.quant_portion_workspace_bytes(pages, entries, heads, dim, page, dtype)
        one = ops._quant_portion(pages, pages, entries, 1, dim, page, dt, 1 << 60)[1]
        assert room <= max(ops.QUANT_PORTION_BYTES, one)
        for n in {1, pages // 3 or 1, pages - 1 or 1, pages}:
            for records in (1, entries):
                h, size = ops._quant_portion(n, pages - n, records, heads, dim, page, dt, room)
                assert 1 <= h <= heads and size <= room
                # 16 bits for every number of the pages of so many heads
                assert size >= n * page * h * dim * 4
                whole = ops._quant_portion(n, pages - n, records, heads, dim, page, dt, 1 << 60)
                assert whole[0] == heads and (h == heads or whole[1] > room)


def test_workspaces_refused():
    cache, t = ops.quant_kv_pool(4, 16, 2, 64, 32, device="cpu"), torch.zeros(8, dtype=torch.int32)
    q, work = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(1, 8, dtype=torch.int32)
    base = dict(q_heads=4, kv_heads=2, head_dim=64, page_size=16)
    room = torch.zeros(4096, dtype=torch.uint8)
    start = -room.data_ptr() % 256
    for bad in (room.to(torch.int32), room[start + 8:], room[::2], room.float()):
        with pytest.raises(ValueError, match="workspace"):
            ops.attn_prefill_paged(q, cache, t, work, workspace=bad, **base)
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.attn_prefill_paged(q, cache, t, work, workspace=room[start:], **base)
