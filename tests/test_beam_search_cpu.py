"""The host's part of a beam search, on a small table of probabilities: candidates from the plain form, against all continuations there are."""
import itertools
import math

import pytest
import torch

import beams_plain as plain
from blitz_scale_b200.runtime.beams import BeamHistory, Candidates


def _search(logits, first, beams, budget, ended, penalty):
    """Continuations of a model whose next logits depend on the last token alone."""
    h, scores, last = BeamHistory(beams, ended, penalty, budget), [0.0], [first]
    for _ in range(budget):
        rows = len(last)
        best, on, _ = plain.select(logits[torch.tensor(last)], torch.tensor(scores), rows, beams * (1 + max(1, len(ended))), beams, set(ended))
        step = Candidates(*([c for c in x[0] if c[1] >= 0] for x in (best, on)))
        h.take(step)
        if h.done:
            break
        scores, last = [c[0] for c in step.next], [c[2] for c in step.next]
    h.close()
    return h.finished


def _all(logits, first, budget, ended):
    """(log probability, tokens, ended) of every continuation."""
    p, out = torch.log_softmax(logits.double(), 1), []
    for n in range(1, budget + 1):
        for t in itertools.product(range(logits.shape[0]), repeat=n):
            stops = t[-1] in ended
            if any(x in ended for x in t[:-1]) or (n < budget and not stops):
                continue
            out.append((sum(p[a, b].item() for a, b in zip((first, *t), t)), list(t), stops))
    return sorted(out, reverse=True)


@pytest.mark.parametrize("seed,ended", [(0, [0]), (1, [0]), (2, [0, 3]), (3, []), (4, [2])])
def test_wide_searches_find_the_best(seed, ended):
    logits = 2 * torch.randn(4, 4, generator=torch.Generator().manual_seed(seed))
    want = _all(logits, 1, 4, set(ended))
    got = _search(logits, 1, 64, 4, ended, 0.0)          # (as many beams as there are continuations of three tokens: nothing is left out)
    assert len(got) == min(64, len(want))
    for h, (p, tokens, stops) in zip(got[:20], want):
        assert abs(h.log_prob - p) < 1e-5 and h.score == h.log_prob
    assert {(tuple(h.tokens), h.ended) for h in got[:5]} == {(tuple(t), s) for _, t, s in want[:5]}


def test_narrow_searches_and_lengths():
    # the first step's best token leads nowhere good; long continuations are worth more with a penalty of one
    logits = torch.full((5, 5), -20.0)
    logits[1, 2], logits[1, 3] = 1.0, 0.9
    logits[2] = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.0])
    logits[3, 4], logits[4, 0] = 10.0, 10.0
    assert _search(logits, 1, 1, 3, [0], 0.0)[0].tokens[0] == 2
    two = _search(logits, 1, 2, 3, [0], 0.0)
    assert two[0].tokens == [3, 4, 0] and two[0].ended
    flat = torch.zeros(3, 3)
    flat[:, 0] = 0.1
    assert _search(flat, 1, 2, 6, [0], 0.0)[0].tokens == [0]
    by_length = _search(flat, 1, 2, 6, [0], 4.0)
    assert len(by_length[0].tokens) == 6 and by_length[0].score == pytest.approx(by_length[0].log_prob / 6 ** 4)


def test_searches_that_end_early():
    logits = torch.full((3, 3), -math.inf)
    logits[1, 0] = 0.0                                    # nothing goes on behind token 0
    got = _search(logits, 1, 4, 5, [0], 1.0)
    assert [(h.tokens, h.log_prob, h.ended) for h in got] == [([0], 0.0, True)]
    h = BeamHistory(2, [0], 1.0, 5)
    h.take(Candidates([], []))
    assert h.done and h.finished == []
    h.close()
    h.take(Candidates([(0.0, 0, 0)], []))
    assert h.finished == []
