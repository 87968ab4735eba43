"""Engine.beam_search: as many beams as selection takes, logits that are no numbers, many shapes, greedy decoding beside one beam, caches full of what others left."""
import pytest
import torch

from blitz_scale_b200.runtime import beams as rb
from blitz_scale_b200.runtime import core
from blitz_scale_b200.runtime.engine import Engine

pytestmark = pytest.mark.gpu


def _prompts(lens, vocab, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (n,), generator=g).tolist() for n in lens]


def _fed(engine, tokens, last):
    """Log probabilities [last, vocab] behind the last `last` prefixes of `tokens`, in one pass over a request of their own."""
    b = engine.new_batch(77, [core.SeqSpec(0, tokens, 1)])
    try:
        return torch.log_softmax(engine.step(b, [len(tokens)], [list(range(len(tokens) - last, len(tokens)))]).double(), 1).cpu()
    finally:
        b.clear()


# Logits of this model are of order one, in bf16: off by 2^-8 each way, and the hidden states behind them by as much again per layer's worth of roundings.
SLACK = 0.06


@pytest.mark.parametrize("beams,eos", [(33, []), (64, []), (32, [5]), (21, [5, 9])])
def test_as_many_beams_as_there_are(beams, eos):
    """beams x (1 + tokens that end a continuation) up to 64."""
    e = Engine("tiny_gpu", num_pages=400, page_size=16, max_batch=64, max_batch_tokens=512)
    prompt = _prompts([20], 4096, seed=8)[0]
    found = e.beam_search([prompt], beams, 5, eos=eos)[0]
    assert len(found) == beams and len({tuple(h.tokens) for h in found}) == beams
    for h in found[:3] + found[-3:]:
        p = _fed(e, prompt + h.tokens[:-1], len(h.tokens))
        assert abs(sum(p[i, t].item() for i, t in enumerate(h.tokens)) - h.log_prob) <= SLACK * len(h.tokens)
    with pytest.raises(ValueError, match=f"at most {64 // (1 + len(eos))} "):
        e.beam_search([prompt], 64 // (1 + len(eos)) + 1, 5, eos=eos)


@pytest.mark.parametrize("after", [0, 3])
def test_logits_that_are_no_numbers(monkeypatch, after):
    e = Engine("tiny_gpu", num_pages=200, page_size=16, max_batch=8, max_batch_tokens=512, use_graphs=False)
    free, forward, calls = e.pool.free_pages, e.runner.forward, []

    def spoilt(meta, **more):
        out = forward(meta, **more)
        if len(calls) == after:
            e.runner.logits[4 if after else 1:].fill_(float("nan"))
        calls.append(meta)
        return out
    monkeypatch.setattr(e.runner, "forward", spoilt)
    with pytest.raises(RuntimeError, match="no numbers"):
        e.beam_search(_prompts([20, 7], 4096, seed=1), 4, 6)
    assert len(calls) == after + 1 and e.pool.free_pages == free
    monkeypatch.undo()
    assert [len(x) for x in e.beam_search(_prompts([20, 7], 4096, seed=1), 4, 6)] == [4, 4]


def test_searches_of_many_shapes(monkeypatch):
    """What is found does not depend on the graphs that came and went before."""
    monkeypatch.setattr(rb, "GRAPHS_MOST", 2)
    e = Engine("tiny_gpu", num_pages=300, page_size=16, max_batch=16, max_batch_tokens=512)
    shapes = [(1, 4, 20), (2, 3, 20), (3, 5, 20), (1, 4, 200), (1, 4, 20), (2, 3, 20), (1, 16, 30)]
    found = []
    for n, beams, length in shapes:
        found.append(e.beam_search(_prompts([length] * n, 4096, seed=length), beams, 8))
        assert len(e._beam_buffers) <= 2 and sum(key[0] == "beams" for key in e._graphs) <= 2
    assert found[0] == found[4] and found[1] == found[5]
