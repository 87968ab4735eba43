"""Beam search's selection at the edges of its definition: rows far from zero, rows of the type's lowest number."""
import math

import pytest
import torch

from blitz_scale_b200 import ops

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32

# What a score may be off by: exponentials to 2^-22, their arguments within 20 of the largest to 20 x 2^-23, about 30 additions in fp32, hence 5e-6 for the log of
# the sum; the score itself is rounded once.
LSE = 5e-6


def _values(z, scores):
    """score + ((z - largest) - log of the sum) in 64 bits, [rows, vocab]: the largest is taken off first, whatever its size."""
    z = z.double().cpu()
    top = z.amax(1, keepdim=True)
    d = z - top
    return scores.double().cpu()[:, None] + (d - d.exp().sum(1, keepdim=True).log())


def _close(got, want):
    """Scores of the candidates in `got` beside the values [requests, beams * vocab] in `want`; no better candidate is left out."""
    Q, n = got.score.shape
    V = want.shape[1]
    best = torch.sort(want.view(Q, -1), dim=1, descending=True).values
    score, parent, token = got.score.double().cpu(), got.parent.tolist(), got.token.tolist()
    of = want.view(Q, -1, V)
    for q in range(Q):
        assert len(set(zip(parent[q], token[q]))) == n
        for i in range(n):
            v = of[q, parent[q][i], token[q][i]].item()
            assert abs(score[q, i].item() - v) <= LSE + 2.0 ** -24 * abs(v), (q, i, score[q, i].item(), v)
            assert v >= best[q, i].item() - 2 * LSE, (q, i, v, best[q, i].item())


@pytest.mark.parametrize("V", [40, 1001, 40001])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_rows_of_the_lowest_number(dtype, V):
    """A row that is masked everywhere: its tokens share its probability, and another beam's likely tokens come before them."""
    z = torch.randn(4, V, generator=torch.Generator("cuda").manual_seed(V), device="cuda")
    z[0] = z[3] = torch.finfo(dtype).min
    z[1, 7], z[2, 3] = 30.0, 30.0
    z = z.to(dtype)
    scores = torch.tensor([-1.0, -1.0, -0.5, -9.0], device="cuda")
    got = ops.beam_select(z, scores, 2, n=8)
    ops.check_status()
    _close(got, _values(z, scores))
    assert (got.parent[0, 0].item(), got.token[0, 0].item()) == (1, 7) and (got.parent[1, 0].item(), got.token[1, 0].item()) == (0, 3)
    alone = ops.beam_select(z[:1], scores[:1], 1, n=8)
    assert alone.token.tolist() == [list(range(8))]
    assert (alone.score.double().cpu() - (-1.0 - math.log(V))).abs().max() <= LSE + 2.0 ** -24 * 20


@pytest.mark.parametrize("offset", [3e3, 1e6, -1e9, 1e20, -1e30, 3e38])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_far_from_zero(dtype, offset):
    """Rows of one large number but for some tokens masked by minus infinity or the type's lowest number."""
    g = torch.Generator("cuda").manual_seed(1)
    z = torch.full((6, 5001), offset, device="cuda")
    z[1::2, torch.rand(5001, generator=g, device="cuda") < 0.5] = -math.inf
    z[2:4, torch.rand(5001, generator=g, device="cuda") < 0.3] = torch.finfo(dtype).min
    z = z.to(dtype)
    scores = torch.tensor([-1.0, -2.0, -0.25, -0.5, -7.0, -3.0], device="cuda")
    got = ops.beam_select(z, scores, 3, n=9)
    ops.check_status()
    _close(got, _values(z, scores))


@pytest.mark.parametrize("dtype", [F32])
def test_rows_of_distances_far_from_zero(dtype):
    """Logits behind a large offset that fp32 still tells apart (steps of 2^-4 around 2^19)."""
    g = torch.Generator("cuda").manual_seed(2)
    z = torch.round(torch.randn(6, 30011, generator=g, device="cuda") * 16) / 16 + float(1 << 19)
    z[1::2] = -z[1::2]
    scores = torch.tensor([-1.0, -2.0, -0.25, -0.5, -7.0, -3.0], device="cuda")
    got = ops.beam_select(z, scores, 2, n=16)
    ops.check_status()
    _close(got, _values(z, scores))
