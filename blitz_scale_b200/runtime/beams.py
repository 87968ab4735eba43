"""Beam search on one GPU: `Engine.beam_search`.

A request's beams are consecutive rows of a decode step and share the pages of what they have in common: prompts from the start, later whatever
the beams that are left come from.  Between two steps the GPU selects, hands out pages, copies the partly filled ones that two beams would write and makes
the next step's tables (`ops.beam_select`, `beam_fork`, `copy_pages`, `step_tables`); the host reads the candidates, keeps the
finished ones and launches the next step, a CUDA graph.  States of recurrent layers move with their beams in the same way, slot by slot.

The reference serves greedily only (src/kernel/sampler.cu:7-141); this is an addition to its interface.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Dict, List, NamedTuple, Optional, Sequence, Tuple

import torch

from .. import ops
from ..models.llama import StepMeta
from . import core


@dataclass
class Hypothesis:
    """A continuation: its tokens (the one that ends it among them), the sum of their log probabilities, what it is ranked by, and whether such a token ended
    it (else the budget did)."""
    tokens: List[int]
    log_prob: float
    score: float
    ended: bool


class Candidates(NamedTuple):
    """A step's candidates of one request, best first, and those that go on, as lists of (score, parent, token); places without one are left out."""
    best: List[Tuple[float, int, int]]
    next: List[Tuple[float, int, int]]


class BeamHistory:
    """One request's search on the host: where every beam of every step came from, and the finished continuations.

    Finished ones are ranked by log probability / length ^ length_penalty; a candidate that ends counts if it is among the first `beams` of its step.
    The search is over when `beams` have finished and no running one can rise above the worst of them: log probabilities only fall, and
    with a penalty above zero the budget's length is the best a running one can have."""

    def __init__(self, beams: int, ended: Sequence[int], length_penalty: float, budget: int):
        self.beams, self.ended, self.penalty, self.budget = beams, frozenset(ended), length_penalty, budget
        self.steps: List[List[Tuple[float, int, int]]] = []
        self.finished: List[Hypothesis] = []
        self.done = False

    def tokens(self, beam: int) -> List[int]:
        """Tokens of a beam of the last step."""
        out = []
        for step in reversed(self.steps):
            _, parent, token = step[beam]
            out.append(token)
            beam = parent
        return out[::-1]

    def _add(self, tokens: List[int], log_prob: float, ended: bool) -> None:
        self.finished.append(Hypothesis(tokens, log_prob, log_prob / len(tokens) ** self.penalty, ended))
        self.finished.sort(key=lambda h: -h.score)
        del self.finished[self.beams:]

    def take(self, step: Candidates) -> None:
        if self.done:
            return
        for score, parent, token in step.best[:self.beams]:
            if token in self.ended:
                self._add((self.tokens(parent) if self.steps else []) + [token], score, True)
        self.steps.append(step.next)
        if not step.next:
            self.done = True
        elif len(self.finished) >= self.beams:
            length = self.budget if self.penalty > 0 else len(self.steps)
            self.done = self.finished[-1].score >= step.next[0][0] / length ** self.penalty

    def close(self) -> None:
        """The budget is spent: what still runs is finished too."""
        if not self.done and self.steps:
            for b, (score, _, _) in enumerate(self.steps[-1]):
                self._add(self.tokens(b), score, False)
        self.done = True


class _Buffers:
    """What a captured step reads and writes, for `rows` rows of up to `width` pages."""

    def __init__(self, rows: int, beams: int, width: int, device):
        new = lambda *s: torch.zeros(*s, dtype=torch.int32, device=device)  # noqa: E731
        self.ids, self.seq_slot = new(rows), new(rows)
        self.tables = ops.StepTables(new(rows * width), new(rows + 1), new(rows), new(rows), new(rows), None, new(rows // beams))


GRAPHS_MOST = 16      # shapes of steps that an engine keeps a graph and buffers for


def _buffers(engine, key: tuple, rows: int, beams: int, width: int) -> _Buffers:
    """The buffers of steps of one shape.  Those that were not used for the longest time make room for a new one, their graph with them.  (No step is under way.)"""
    kept = engine._beam_buffers        # (the last used one is the last)
    buf = kept.pop(key, None)
    if buf is None:
        while len(kept) >= GRAPHS_MOST:
            old = next(iter(kept))
            engine._graphs.pop(old, None)
            del kept[old]
        buf = _Buffers(rows, beams, width, engine.device)
    kept[key] = buf
    return buf


def _graph_rows(groups: int, beams: int, most: int) -> int:
    """Groups of a step: the next power of two, where the engine's batch has room for it (steps of similar batches share a graph)."""
    n = 1
    while n < groups:
        n *= 2
    return n if n * beams <= most else groups


def _tensors(engine) -> Tuple[list, list]:
    """(caches whose pages are copied, as arguments of ops.copy_pages; state tensors [slots, ...])"""
    if engine.cfg.family != "hybrid":
        return [(engine.kv, True)], []
    pools, states, seen = [], [], set()
    for run in engine.cache.runs:
        if run.kv is not None and id(run.kv) not in seen:
            seen.add(id(run.kv))
            pools.append((run.kv, False))
        states += [t for t in (run.state, run.hist, run.mix_hist, run.shift) if t is not None and t.numel()]
    return pools, states


class _Search:
    """One batch of requests, beams x requests <= max_batch."""

    def __init__(self, engine, prompts: Sequence[Sequence[int]], beams: int, budget: int, ended: Sequence[int], length_penalty: float):
        self.e, self.beams, self.budget, self.Q = engine, beams, budget, len(prompts)
        self.lens = [len(p) for p in prompts]
        self.history = [BeamHistory(beams, ended, length_penalty, budget) for _ in prompts]
        self.n = min(ops.BEAMS_MAX, beams * (1 + max(1, len(ended))))        # (so many of them may end that this is what leaves `beams`)
        dev = engine.device
        self.ended = torch.tensor(list(ended), dtype=torch.int32, device=dev) if len(ended) else None
        specs = [core.SeqSpec(i, list(map(int, p)), 1) for i, p in enumerate(prompts)]
        self.batch, self.pages, self.slots = None, [], []
        try:
            self._reserve(specs)
        except Exception:
            self.release()
            raise

    def _reserve(self, specs) -> None:
        """The prompts' pages, and for every beam those that it may come to have for itself; a state slot for every beam."""
        e, ps = self.e, self.e.page_size
        self.batch = e.new_batch((1 << 62) + 1, specs)
        if self.batch is None:
            raise RuntimeError("the cache has too few free pages or state slots for the prompts")
        self.pool, self.slot_pool = [], []
        for seq, n in zip(self.batch.seqs, self.lens):
            own = -(-(n + self.budget) // ps) - n // ps
            more = e.pool.allocate(max(0, n // ps + self.beams * own - len(seq.pages)))
            if more is None:
                raise RuntimeError(f"the cache has too few free pages for {self.beams} beams of {n} + {self.budget} tokens")
            self.pages += more
            self.pool.append(list(seq.pages) + more)
            if e.slots is not None:
                got = [seq.slot]
                for _ in range(self.beams - 1):
                    s = e.slots.allocate()
                    if s < 0:
                        raise RuntimeError(f"too few free state slots for {self.beams} beams")
                    self.slots.append(s)
                    got.append(s)
                self.slot_pool.append(got)
        self.width = max(-(-(n + self.budget) // ps) for n in self.lens) + 1

    def release(self) -> None:
        if self.batch is not None:
            self.batch.clear()
        if self.pages:
            self.e.pool.release(self.pages)
        for s in self.slots:
            self.e.slots.release(s)
        self.batch, self.pages, self.slots = None, [], []

    # ------------------------------------------------------------------ one step
    def _at_once(self) -> bool:
        """Whether the cache is one that attention reads once for a request's beams; others go through attn_decode, row by row."""
        e, ps = self.e, self.e.page_size
        return e.cfg.family != "hybrid" and e.kv_bits == 16 and e.cfg.head_dim in (64, 128) and ps >= 16 and ps & (ps - 1) == 0

    def _step_meta(self, rows: int, buf: _Buffers, splits: int) -> StepMeta:
        t = buf.tables
        shared = t.shared if self._at_once() else None
        return StepMeta(ids=buf.ids, pos=t.pos, slot=t.slot, page_indices=t.indices, page_indptr=t.indptr, last_page_len=t.last_page_len, seq_slot=buf.seq_slot,
                        batch=rows, num_tokens=rows, num_splits=splits, static_positions=True, beams=self.beams, shared=shared)

    def _forward(self, rows: int, buf: _Buffers, splits: int, key: tuple) -> None:
        """A decode step over the buffers' rows.  (The stream is idle: nothing that writes the tables is still running.)"""
        e = self.e
        meta = self._step_meta(rows, buf, splits)
        if not e.use_graphs:
            e.runner.forward(meta)
            return
        g = e._graphs.get(key)
        if g is None:
            # (warm-up outside the capture; rows without a slot, so that no cache row and no state is written)
            keep = [t.clone() for t in (buf.tables.slot, buf.seq_slot)]
            buf.tables.slot.fill_(-1)
            buf.seq_slot.fill_(-1)
            torch.cuda.current_stream().synchronize()
            e.runner.forward(meta)
            for t, v in zip((buf.tables.slot, buf.seq_slot), keep):
                t.copy_(v)
            torch.cuda.current_stream().synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, capture_error_mode="thread_local"):
                e.runner.forward(meta)
            e._graphs[key] = g
        g.replay()

    @torch.no_grad()
    def run(self) -> List[List[Hypothesis]]:
        e, Q, k, n = self.e, self.Q, self.beams, self.n
        dev, ps = e.device, e.page_size
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        e.prefill(self.batch)
        groups = _graph_rows(Q, k, e.max_batch)
        rows, width = groups * k, 1 << (self.width - 1).bit_length()
        longest = max(self.lens) + self.budget
        splits = 1 if self._at_once() else e.choose_splits(Q * k, longest, sum(self.lens) * k + Q * k * self.budget)
        key = ("beams", rows, k, width, splits)
        buf = _buffers(e, key, rows, k, width)
        pools, states = _tensors(e)
        # the request's rows before its first step: one, with the prompt
        pad = lambda x, m: x + [-1] * (m - len(x))  # noqa: E731
        table = i32([pad(list(s.pages)[:-(-m // ps)], width) for s, m in zip(self.batch.seqs, self.lens)])
        cached = i32(self.lens)
        most = max(len(p) for p in self.pool)
        pool = i32([pad(p, most) for p in self.pool])
        if e.slots is not None:
            slot_table, one = i32([[p[0]] for p in self.slot_pool]), i32([1] * Q)
            slot_pool = i32(self.slot_pool)
        # a step's candidates lie one behind the other, so that one copy brings them
        flat = torch.empty(3 * Q * (n + k), dtype=torch.float32, device=dev)
        host = torch.empty(flat.shape, dtype=torch.float32, pin_memory=True)
        cuts = [Q * n] * 3 + [Q * k] * 3

        def parts(t):
            p = t.split(cuts)
            return [p[0], p[1].view(torch.int32), p[2].view(torch.int32), p[3], p[4].view(torch.int32), p[5].view(torch.int32)]
        got = ops.BeamStep(*(x.view(Q, n if i < 3 else k) for i, x in enumerate(parts(flat))))
        scores = torch.zeros(Q, dtype=torch.float32, device=dev)
        full_table = torch.full((rows, width), -1, dtype=torch.int32, device=dev)
        full_cached = torch.full((rows,), -1, dtype=torch.int32, device=dev)
        buf.ids.zero_()
        buf.seq_slot.fill_(-1)
        for step in range(self.budget):
            ops.beam_select(e.runner.logits[:Q * (k if step else 1)], scores, k if step else 1, n=n, keep=k, ended=self.ended, out=got)
            last = step + 1 == self.budget
            if not last:
                scores = got.next_score.reshape(-1).clone()
                fork = ops.beam_fork(table, cached, got.next_parent, pool, page_size=ps, num_pages=e.num_pages)
                for cache, layers in pools:
                    tokens = fork.tokens if e.kv_bits == 16 else None
                    ops.copy_pages(cache, fork.src, fork.dst, tokens, layers=layers)
                if e.slots is not None:
                    slots = ops.beam_fork(slot_table, one, got.next_parent, slot_pool, page_size=2, num_pages=e.cache.num_slots)
                    for t in states:
                        ops.copy_pages(t, slots.src, slots.dst)
                    slot_table, one = slots.table, slots.cached
                    buf.seq_slot[:Q * k].copy_(slot_table.view(-1))
                table, cached = fork.table, fork.cached
                full_table[:Q * k].copy_(table)
                full_cached[:Q * k].copy_(cached)
                ops.step_tables(full_table, full_cached, page_size=ps, beams=k, out=buf.tables)
                buf.ids[:Q * k].copy_(got.next_token.view(-1).clamp(min=0))
                cached = torch.where(cached >= 0, cached + 1, cached)       # (with the token that the step will write)
            host.copy_(flat, non_blocking=True)
            torch.cuda.current_stream().synchronize()
            self._note(parts(host))
            over = [q for q, h in enumerate(self.history) if h.done]
            if last or len(over) == Q:
                break
            if over:        # nothing goes on from there: their rows are dead from the next selection on
                scores.view(Q, k)[over] = -float("inf")
            self._forward(rows, buf, splits, key)
        ops.check_status(dev)
        for h in self.history:
            h.close()
        return [h.finished for h in self.history]

    def _note(self, p: List[torch.Tensor]) -> None:
        """Takes a step's candidates into the requests' histories."""
        p = [x.tolist() for x in p]
        for q, h in enumerate(self.history):
            lists = [[(p[i][j], p[i + 1][j], p[i + 2][j]) for j in range(q * m, q * m + m) if p[i + 1][j] >= 0] for i, m in ((0, self.n), (3, self.beams))]
            if not h.done and not lists[0]:
                raise RuntimeError("beam search: the logits of a request are no numbers (NaN or infinity)")
            h.take(Candidates(*lists))


def beam_search(engine, prompts: Sequence[Sequence[int]], beams: int, max_new_tokens: int, *, eos: Sequence[int] = (), length_penalty: float = 1.0,
                best: Optional[int] = None) -> List[List[Hypothesis]]:
    """See Engine.beam_search."""
    if engine.tp > 1:
        raise RuntimeError("beam search runs on one GPU")
    if not engine.status.fully_loaded():
        raise RuntimeError("model parameters are not loaded")
    eos = sorted({int(t) for t in eos})
    most = min(ops.BEAMS_MAX // (1 + len(eos)), engine.max_batch)
    if not 1 <= beams <= most:
        raise ValueError(f"{beams} beams: at most {most} with {len(eos)} tokens that end a continuation, {ops.BEAMS_MAX} candidates and max_batch={engine.max_batch}")
    try:
        longest = float(max_new_tokens) ** length_penalty if max_new_tokens > 0 else 1.0
    except OverflowError:
        longest = math.inf
    if not 0.0 < longest < math.inf or (best is not None and best < 1):
        raise ValueError(f"a length penalty of {length_penalty} over {max_new_tokens} tokens, the best {best}")
    if max_new_tokens < 1 or any(len(p) < 1 for p in prompts):
        raise ValueError("a prompt of one token and a budget of one at least")
    if not all(0 <= t < engine.cfg.vocab for p in (eos, *prompts) for t in p):
        raise ValueError(f"tokens of a vocabulary of {engine.cfg.vocab}")
    per, out = max(1, engine.max_batch // beams), []
    for i in range(0, len(prompts), per):
        search = _Search(engine, prompts[i:i + per], beams, max_new_tokens, eos, length_penalty)
        try:
            out += search.run()
        finally:
            torch.cuda.current_stream().synchronize()
            search.release()
    return [h[:best] for h in out]
