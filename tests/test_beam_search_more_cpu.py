"""The host's part of a beam search: requests without candidates, what is kept between searches, refusals."""
import math

import pytest
import torch

from blitz_scale_b200.runtime import beams as rb


def _search(Q, beams, n):
    s = rb._Search.__new__(rb._Search)
    s.Q, s.beams, s.n = Q, beams, n
    s.history = [rb.BeamHistory(beams, [0], 1.0, 5) for _ in range(Q)]
    return s


def _step(*rows):
    """Candidates as they come from the GPU: for each request `best` and `next`, lists of (score, parent, token)."""
    return [torch.tensor([c[i] for row in rows for c in row[j]], dtype=torch.float32 if i == 0 else torch.int32) for j in (0, 1) for i in range(3)]


NONE = (-math.inf, -1, -1)


def test_requests_without_candidates():
    """A running request without any candidate is an error, one that is over has none."""
    s = _search(2, 2, 4)
    s._note(_step(([(-1.0, 0, 3), (-2.0, 0, 4), NONE, NONE], [(-1.0, 0, 3), (-2.0, 0, 4)]), ([(-1.0, 0, 0), NONE, NONE, NONE], [NONE, NONE])))
    assert not s.history[0].done and s.history[1].done and [h.tokens for h in s.history[1].finished] == [[0]]
    s._note(_step(([(-1.5, 1, 3), NONE, NONE, NONE], [(-1.5, 1, 3), NONE]), ([NONE] * 4, [NONE] * 2)))
    assert s.history[0].tokens(0) == [4, 3]
    with pytest.raises(RuntimeError, match="no numbers"):
        s._note(_step(([NONE] * 4, [NONE] * 2), ([NONE] * 4, [NONE] * 2)))


def test_shapes_that_are_kept(monkeypatch):
    """Graphs and buffers of the last used shapes of steps, dropped together; other graphs of the engine stay."""
    monkeypatch.setattr(rb, "_Buffers", lambda *shape: shape)
    monkeypatch.setattr(rb, "GRAPHS_MOST", 3)

    class engine:
        device, _beam_buffers, _graphs = "cpu", {}, {(8, 1): "decode"}
    for i in (1, 2, 3, 1, 4, 1, 5, 5, 2):
        assert rb._buffers(engine, ("beams", i), i, 1, 2) == (i, 1, 2, "cpu")
        engine._graphs[("beams", i)] = i
        assert len(engine._beam_buffers) <= 3
    assert list(engine._beam_buffers) == [("beams", i) for i in (1, 5, 2)]
    assert engine._graphs == {(8, 1): "decode", ("beams", 1): 1, ("beams", 5): 5, ("beams", 2): 2}


class _Engine:
    """As much of an engine as the checks of arguments look at."""
    tp, max_batch = 1, 8

    class status:
        fully_loaded = staticmethod(lambda: True)

    class cfg:
        vocab = 100


@pytest.mark.parametrize("more", [dict(best=0), dict(best=-1), dict(length_penalty=math.nan), dict(length_penalty=math.inf), dict(length_penalty=-math.inf), dict(length_penalty=1e4),
                                  dict(length_penalty=-1e4)])
def test_refusals(more):
    with pytest.raises(ValueError, match="length penalty"):
        rb.beam_search(_Engine(), [[1, 2]], 4, 20, **more)
    assert rb.beam_search(_Engine(), [], 4, 20, length_penalty=-2.0, best=1) == []
