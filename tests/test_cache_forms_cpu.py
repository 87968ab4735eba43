"""Replicas of a cluster have caches of one form: those of others are refused when the workers start, and the router counts its bytes."""
import multiprocessing

import pytest


def _rank(rank, world, store, form, queue):
    import torch.distributed as dist
    from blitz_scale_b200.parallel.agreement import same_on_all_ranks
    dist.init_process_group("gloo", init_method=f"file://{store}", rank=rank, world_size=world)
    try:
        queue.put((rank, same_on_all_ranks("the cache's form", form)))
    except ValueError as e:
        queue.put((rank, str(e)))
    dist.barrier()
    dist.destroy_process_group()


def _backend(rank, world, store, more, queue):
    """A worker's set-up up to its first memory."""
    import torch
    import torch.distributed as dist
    dist.init_process_group("gloo", init_method=f"file://{store}", rank=rank, world_size=world)
    torch.cuda.current_device = lambda: 0
    from blitz_scale_b200.parallel import symm
    from blitz_scale_b200.worker.gpu_backend import GpuBackend

    class Reached(Exception):
        pass

    def fabric(*a, **k):
        raise Reached
    symm.PeerFabric = fabric
    try:
        GpuBackend(rank, world, "tiny", **more)
    except ValueError as e:
        queue.put((rank, str(e)))
    except Reached:
        queue.put((rank, "the same"))
    dist.barrier()
    dist.destroy_process_group()


def _run(target, values, tmp_path):
    ctx = multiprocessing.get_context("spawn")
    queue, store = ctx.Queue(), tmp_path / "store"
    procs = [ctx.Process(target=target, args=(r, len(values), str(store), v, queue)) for r, v in enumerate(values)]
    for p in procs:
        p.start()
    out = dict(queue.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    return [out[r] for r in range(len(values))]


def test_forms_are_compared(tmp_path):
    a = {"kv_bits": 4, "kv_group": 32}
    assert _run(_rank, [a, dict(a)], tmp_path) == [a, a]


@pytest.mark.parametrize("more", [dict(kv_bits=16), dict(kv_bits=4, kv_group=32), dict(kv_bits=4, kv_group=64, page_size=32)])
def test_workers_of_another_form_do_not_start(tmp_path, more):
    said = _run(_backend, [dict(kv_bits=4, kv_group=64), more], tmp_path)
    for s in said:
        assert "cache's form differs between ranks" in s and "'kv_bits': 4" in s and f"'kv_bits': {more['kv_bits']}" in s


def test_workers_of_one_form_start(tmp_path):
    assert _run(_backend, [dict(kv_bits=4, kv_group=32)] * 2, tmp_path) == ["the same"] * 2


def test_groups_do_not_matter_to_a_16_bit_cache(tmp_path):
    assert _run(_backend, [dict(kv_bits=16, kv_group=32), dict(kv_bits=16, kv_group=64)], tmp_path) == ["the same"] * 2


@pytest.mark.parametrize("group", [32, 64, 128])
def test_bytes_of_a_migrated_token(group):
    from blitz_scale_b200.models.config import get_config
    from blitz_scale_b200.router.server import build_parser, kv_mb_per_token
    from blitz_scale_b200.runtime.engine import kv_page_bytes
    c = get_config("llama3_8b")
    a = build_parser().parse_args(["--kv-bits", "4", "--kv-group", str(group), "--client-config", "[]", "--deployment-config-path", "x"])
    assert kv_mb_per_token(c, a.kv_bits, a.kv_group) * 1e6 == pytest.approx(c.layers * kv_page_bytes(c, 64, kv_bits=4, kv_group=group) / 64)
    a = build_parser().parse_args(["--client-config", "[]", "--deployment-config-path", "x"])
    assert kv_mb_per_token(c, a.kv_bits, a.kv_group) * 1e6 == pytest.approx(c.kv_bytes_per_token())
