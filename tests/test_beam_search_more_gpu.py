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


def test_one_beam_takes_what_greedy_decoding_takes():
    """Token by token, up to one where the two largest logits are nearer than what two ways of computing them differ by."""
    e = Engine("tiny_gpu", num_pages=200, page_size=16, max_batch=8, max_batch_tokens=512)
    for prompt in _prompts([30, 1, 64, 15, 100], 4096, seed=2):
        batch = e.new_batch(1, [core.SeqSpec(0, prompt, 12)])
        greedy = [t for step in [e.prefill(batch)] + [e.decode(batch) for _ in range(11)] for t in step]
        batch.clear()
        found = e.beam_search([prompt], 1, 12)[0]
        assert len(found) == 1 and len(found[0].tokens) == 12
        same = next((i for i, (a, b) in enumerate(zip(greedy, found[0].tokens)) if a != b), 12)
        if same < 12:
            p = _fed(e, prompt + greedy[:same], 1)[0]
            assert abs(p[greedy[same]] - p[found[0].tokens[same]]) <= 2 * SLACK


@pytest.mark.parametrize("page,lens,beams", [(16, [1, 16, 33, 47], 4), (64, [5, 64, 130], 5)])
def test_caches_full_of_what_others_left(page, lens, beams):
    """Pages that no request has written hold large numbers: a token that a copy leaves out, or a page taken for another, would take all the weight.  What is
    found is what an empty cache gives, to the last bit."""
    e = Engine("tiny_gpu", num_pages=200, page_size=page, max_batch=32, max_batch_tokens=512)
    prompts = _prompts(lens, 4096, seed=9)
    found = []
    for left in (0.0, 100.0, -3.0):
        e.kv.fill_(left)
        found.append(e.beam_search(prompts, beams, 2 * page + 3 if page == 16 else 70))
    assert found[0] == found[1] == found[2]
