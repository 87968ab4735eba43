"""Engine.beam_search: every step's choice beside the logits that the beams' tokens have in passes of their own, over caches of each kind."""
import math

import pytest
import torch

from blitz_scale_b200 import ops
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
        z = engine.step(b, [len(tokens)], [list(range(len(tokens) - last, len(tokens)))])
        return torch.log_softmax(z.double(), 1).cpu()
    finally:
        b.clear()


def _checked(engine, prompts, beams, budget, slack, eos=(), monkeypatch=None, **more):
    """A search whose steps are compared with what single passes give: the candidates of a step are the best ones but for `slack`, what the two ways of computing
    a log probability may differ by."""
    seen = []
    take = rb.BeamHistory.take

    def noted(self, step):
        seen.append((self, step, [self.tokens(b) for b in range(len(self.steps[-1]))] if self.steps else [[]], [c[0] for c in self.steps[-1]] if self.steps else [0.0],
                     self.done))
        take(self, step)
    monkeypatch.setattr(rb.BeamHistory, "take", noted)
    free = engine.pool.free_pages, None if engine.slots is None else engine.slots.free_slots
    found = engine.beam_search(prompts, beams, budget, eos=eos, **more)
    assert (engine.pool.free_pages, None if engine.slots is None else engine.slots.free_slots) == free
    histories = []
    for h, *_ in seen:
        if h not in histories:
            histories.append(h)
    assert len(histories) == len(prompts) == len(found)
    for h, prompt, hyps in zip(histories, prompts, found):
        for who, step, tokens, scores, done in seen:
            if who is not h or done:
                continue
            p = torch.stack([_fed(engine, prompt + t, 1)[0] for t in tokens]) + torch.tensor(scores).double()[:, None]
            best = torch.sort(p.flatten(), descending=True).values
            assert len(step.best) == min(len(best), beams * (1 + max(1, len(eos))))
            for i, (score, parent, token) in enumerate(step.best):
                at = p[parent, token].item()
                assert abs(at - score) <= slack and at >= best[i].item() - 2 * slack, (i, at, score, best[i])
            assert step.next == [c for c in step.best if c[2] not in eos][:beams]
        for x in hyps:
            assert len(x.tokens) <= budget and (x.tokens[-1] in eos) == x.ended and (x.ended or len(x.tokens) == budget)
            whole = _fed(engine, prompt + x.tokens[:-1], len(x.tokens)) if len(prompt) + len(x.tokens) > 1 else None
            total = sum(whole[i, t].item() for i, t in enumerate(x.tokens))
            assert abs(total - x.log_prob) <= slack * len(x.tokens)
            assert x.score == pytest.approx(x.log_prob / len(x.tokens) ** more.get("length_penalty", 1.0))
        assert [x.score for x in hyps] == sorted((x.score for x in hyps), reverse=True)
    ops.check_status()
    return found


# Logits of these models are of order one, in bf16: off by 2^-8 each way, and the hidden states behind them by as much again per layer's worth of roundings.
SLACK = 0.06


@pytest.mark.parametrize("use_graphs", [True, False])
@pytest.mark.parametrize("page,lens,beams", [(64, [5, 64, 130], 4), (16, [1, 16, 33, 47], 3)])
def test_uniform_model(monkeypatch, use_graphs, page, lens, beams):
    e = Engine("tiny_gpu", num_pages=200, page_size=page, max_batch=16, max_batch_tokens=512, use_graphs=use_graphs)
    _checked(e, _prompts(lens, 4096), beams, 20, SLACK, monkeypatch=monkeypatch)


@pytest.mark.parametrize("page", [8, 48])
def test_pages_that_attention_of_beams_does_not_take(monkeypatch, page):
    e = Engine("tiny_gpu", num_pages=200, page_size=page, max_batch=16, max_batch_tokens=512)
    prompts, free = _prompts([1, 47, 100], 4096, seed=7), e.pool.free_pages
    if page == 48:        # (nor does the engine's prefill)
        with pytest.raises(RuntimeError, match="not supported"):
            e.beam_search(prompts, 3, 12)
        assert e.pool.free_pages == free
    else:
        _checked(e, prompts, 3, 12, SLACK, monkeypatch=monkeypatch)


def test_searches_that_end(monkeypatch):
    e = Engine("tiny_gpu", num_pages=200, page_size=16, max_batch=16, max_batch_tokens=512)
    prompts = _prompts([20, 7], 4096, seed=1)
    first = e.beam_search(prompts, 4, 6)
    # tokens that beams take become those that end one
    eos = sorted({h.tokens[i] for x in first for h in x[:2] for i in (1, 3)})[:3]
    found = _checked(e, prompts, 4, 12, SLACK, eos=eos, monkeypatch=monkeypatch, length_penalty=0.5)
    assert any(h.ended for x in found for h in x)
    assert [len(x) for x in e.beam_search(prompts, 4, 6, best=1)] == [1, 1]


def test_one_beam_is_greedy(monkeypatch):
    e = Engine("tiny_gpu", num_pages=100, page_size=64, max_batch=8, max_batch_tokens=512)
    found = _checked(e, _prompts([30], 4096, seed=2), 1, 10, SLACK, monkeypatch=monkeypatch)
    assert len(found[0]) == 1 and len(found[0][0].tokens) == 10


def test_more_requests_than_a_batch_holds_and_long_prompts(monkeypatch):
    e = Engine("tiny_gpu", num_pages=400, page_size=16, max_batch=8, max_batch_tokens=128)
    _checked(e, _prompts([300, 3, 40, 41, 5], 4096, seed=3), 4, 6, SLACK, monkeypatch=monkeypatch)
    again = e.beam_search(_prompts([300, 3], 4096, seed=3), 4, 6)
    assert again == e.beam_search(_prompts([300, 3], 4096, seed=3), 4, 6)


def test_cache_in_4_bits(monkeypatch):
    e = Engine("tiny_gpu", num_pages=200, page_size=16, max_batch=16, max_batch_tokens=512, kv_bits=4)
    # (single passes read the same 4-bit numbers: the cache's own error is on both sides)
    _checked(e, _prompts([9, 50], 4096, seed=4), 4, 12, 2 * SLACK, monkeypatch=monkeypatch)


@pytest.mark.parametrize("name", ["fafudra_tiny", "komulorn_tiny", "vofidra_tiny", "norusun_tiny"])
def test_hybrid_models(monkeypatch, name):
    """States of recurrent layers, pools of other shapes, in 32 bits: what a beam has is what it has alone."""
    e = Engine(name, num_pages=120, page_size=16, max_batch=12, max_batch_tokens=512, dtype=torch.float32, state_slots=20)
    _checked(e, _prompts([18, 1, 33], e.cfg.vocab, seed=5), 4, 8, 2e-3, monkeypatch=monkeypatch)


def test_refusals():
    e = Engine("tiny_gpu", num_pages=20, page_size=16, max_batch=8, max_batch_tokens=512)
    free = e.pool.free_pages
    for args in (([[1]], 0, 4), ([[1]], 9, 4), ([[1]], 4, 0), ([[]], 4, 4), ([[4096]], 4, 4), ([[-1]], 4, 4)):
        with pytest.raises(ValueError):
            e.beam_search(*args)
    with pytest.raises(ValueError):
        e.beam_search([[1]], 2, 4, eos=[5000])
    with pytest.raises(ValueError, match="at most 6 with 9"):
        e.beam_search([[1]], 7, 4, eos=range(9))
    assert len(e.beam_search([[1]], 6, 2, eos=[*range(9), *range(9)])[0]) == 6
    with pytest.raises(RuntimeError, match="too few free pages"):
        e.beam_search([[1] * 100], 8, 100)
    with pytest.raises(RuntimeError, match="too few free pages"):
        e.beam_search([[1] * 500], 2, 4)
    assert e.pool.free_pages == free and e.beam_search([], 4, 4) == []
    assert len(e.beam_search([[1, 2, 3]], 8, 4)[0]) == 8
    e.reset_status()
    with pytest.raises(RuntimeError, match="not loaded"):
        e.beam_search([[1]], 2, 2)


def test_prompts_share_pages_with_other_work():
    """A running batch keeps its tokens while searches come and go in the same cache."""
    e = Engine("tiny_gpu", num_pages=120, page_size=16, max_batch=8, max_batch_tokens=512)
    spec = lambda: [core.SeqSpec(9, _prompts([40], 4096, seed=6)[0], 30)]  # noqa: E731
    alone = e.new_batch(1, spec())
    want = [e.prefill(alone)] + [e.decode(alone) for _ in range(12)]
    alone.clear()
    batch = e.new_batch(2, spec())
    got = [e.prefill(batch)]
    for i in range(12):
        if i % 4 == 1:
            e.beam_search(_prompts([15, 20], 4096, seed=i), 4, 9)
        got.append(e.decode(batch))
    batch.clear()
    assert got == want and math.isfinite(sum(sum(x) for x in got))
