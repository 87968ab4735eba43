"""Beam search's selection where candidates of different beams are equal, and rows begin anywhere."""
import math

import pytest
import torch

from blitz_scale_b200 import ops

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("V", [41, 517, 1003, 50257, 128257])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_equal_rows_wherever_they_begin(dtype, V):
    """Beams of equal logits and scores have equal candidates: the lowest beam comes first, whichever boundary its row begins on."""
    g = torch.Generator("cuda").manual_seed(V)
    for beams, start, gap in ((8, 0, 0), (4, 3, 0), (2, 1, 2), (8, 5, 4), (16, 0, 0)):
        n = min(32, 4 * beams)
        pitch = V + gap
        room = torch.full((start + 3 * beams * pitch,), 1000.0, dtype=dtype, device="cuda")
        z = room[start:].view(3 * beams, pitch)[:, :V]
        rows = (3.0 * torch.randn(3, V, generator=g, device="cuda")).to(dtype)
        z.copy_(rows.repeat_interleave(beams, 0))
        got = ops.beam_select(z, torch.full((3 * beams,), -2.5, device="cuda"), beams, n=n)
        ops.check_status()
        for q, row in enumerate(rows.double().cpu().tolist()):
            best = sorted(range(V), key=lambda t: (-row[t], t))[:n]
            want = sorted(((-row[t], b, t) for t in best for b in range(beams)))[:n]
            assert list(zip(got.parent[q].tolist(), got.token[q].tolist())) == [(b, t) for _, b, t in want], (beams, start, gap, q)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_row_s_results_do_not_depend_on_where_it_begins(dtype):
    """The same rows at every place of 16 bytes: all outputs are equal to the last bit."""
    g = torch.Generator("cuda").manual_seed(4)
    rows = (3.0 * torch.randn(12, 30001, generator=g, device="cuda")).to(dtype)
    rows[:, torch.rand(30001, generator=g, device="cuda") < 0.2] = -math.inf
    scores = -5.0 * torch.rand(12, generator=g, device="cuda")
    want = None
    for start in range(16 // rows.element_size() + 1):
        for gap in (0, 1, 7):
            room = torch.full((start + 12 * (30001 + gap),), 1000.0, dtype=dtype, device="cuda")
            z = room[start:].view(12, 30001 + gap)[:, :30001]
            z.copy_(rows)
            got = ops.beam_select(z, scores, 4, n=20)
            want = want or got
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (start, gap)
    ops.check_status()
