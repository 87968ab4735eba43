"""Beam search over a paged cache: entry points of csrc/kernels/beam.cu and attn_beams.cu.

A request's beams are `beams` consecutive rows.  A row's table names its pages; rows of a request share pages that are full, and of a partly
filled page each has its own.  A step: `attn_decode_beams` in every layer, `beam_select` on the logits, `beam_fork` for the tables of
the beams that go on, `copy_pages` for what two of them cannot share, `step_tables` for the next step's inputs.  Everything stays on the GPU
and can be captured into a graph.  Outputs that a caller gives (`out`) share no memory with the inputs.
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional, Union

import torch

from . import _DT, _DT3, KVPair, LatentKV, QuantKV, _check, _int32, _quant, _raw_device, _status_ptr, _stream
from ._lib import lib

BEAMS_MAX = 64      # beams of a request, and candidates of it


class BeamStep(NamedTuple):
    """The best continuations of every request, [requests, n], best first: score, the beam it comes from and its token (-inf, -1 and -1 where there
    is none); and those that go on, [requests, keep]: the first ones whose token does not end a sequence.  (Where `beam_select` makes them, the first three
    are columns of one tensor.)"""
    score: torch.Tensor
    parent: torch.Tensor
    token: torch.Tensor
    next_score: torch.Tensor
    next_parent: torch.Tensor
    next_token: torch.Tensor


class BeamFork(NamedTuple):
    """Tables of the children [requests * children, width] (-1 behind a row's last page), the tokens they hold (-1: a dead row), and for each the
    copy it asks for: page `src` to page `dst`, `tokens` of them (-1, -1 and 0: none)."""
    table: torch.Tensor
    cached: torch.Tensor
    src: torch.Tensor
    dst: torch.Tensor
    tokens: torch.Tensor


class StepTables(NamedTuple):
    """What a step's kernels read: pages of all rows one behind the other, where each row's begin, tokens on its last page, positions and slots of the
    new tokens; where each row's tokens begin (with counts), and how many pages each request's rows have in common (with beams)."""
    indices: torch.Tensor
    indptr: torch.Tensor
    last_page_len: torch.Tensor
    pos: torch.Tensor
    slot: torch.Tensor
    tok_indptr: Optional[torch.Tensor]
    shared: Optional[torch.Tensor]


def _here(t: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    """All tensors are on the current device."""
    at = t.get_device()
    if at < 0 or at != _raw_device():
        raise ValueError(f"a tensor on {t.device}: the kernels run on the current CUDA device")
    for o in others:
        if not (o is None or o.get_device() == at):
            raise ValueError(f"a tensor on {o.device}, another on {t.device}: the kernels run on the current CUDA device")


def _ints(t: torch.Tensor, shape: tuple, what: str) -> torch.Tensor:
    if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what}: contiguous int32 {tuple(shape)}, got {tuple(t.shape)} {t.dtype}")
    return t


def _numbers(t: torch.Tensor, n: int, what: str) -> None:
    if t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{what}: {n} int32 numbers, got {tuple(t.shape)} {t.dtype}")


def _rows_of(t: torch.Tensor, what: str) -> tuple:
    """(rows, columns, pitch) of a table of int32"""
    shape, step = t.shape, t.stride()
    if t.dtype is not torch.int32 or len(shape) != 2 or (shape[1] > 1 and step[1] != 1):
        raise ValueError(f"{what}: rows of int32, got {tuple(shape)} {t.dtype}")
    return shape[0], shape[1], step[0]


@lru_cache(256)
def _select_scratch(rows: int, vocab: int, n: int, dt: int, device: int) -> int:
    """Scratch of a selection on the current device, in 32-bit words."""
    return (lib().blitz_beam_select_workspace_bytes(rows, vocab, n, dt) + 3) // 4


@lru_cache(256)
def _attn_scratch(rows: int, beams: int, q_heads: int, kv_heads: int, head_dim: int, device: int) -> int:
    return int(lib().blitz_attn_beams_workspace_bytes(rows, beams, q_heads, kv_heads, head_dim))


def beam_select(logits: torch.Tensor, scores: torch.Tensor, beams: int = 1, *, n: int = 0, keep: int = 0, ended: Optional[torch.Tensor] = None,
                out: Optional[BeamStep] = None) -> BeamStep:
    """The ``n`` (2 beams) best continuations of every request.  ``logits`` [requests * beams, vocab] in fp16, bf16 or fp32, rows of any pitch;
    ``scores`` [requests * beams] in fp32, finite, or -inf for a row that has ended.  A continuation's value is the row's score plus the token's log
    probability, a softmax over the whole row; one that is no number (rows with a NaN or +inf), or below what fp32 holds, counts as -inf.  Ties go to the lowest beam, then the
    lowest token: tokens of equal logits in a row, and beams of equal logits and scores, wherever in memory their rows begin.  (A row's log probabilities are off by 5e-6
    at most, all alike: candidates of rows with other logits that are nearer than that may come in either order.)  ``ended``: int32 tokens that end a sequence; ``keep`` (beams): how many continuations go on.  At most 64 beams and candidates."""
    dt = _DT3.get(logits.dtype)
    if dt is None:
        raise TypeError(f"kernel takes fp16/bf16/fp32 tensors, got {logits.dtype}")
    shape, step = logits.shape, logits.stride()
    if len(shape) != 2 or shape[1] < 1 or (step[1] != 1 and shape[1] > 1):
        raise ValueError(f"logits: rows of numbers, got {tuple(shape)}, strides {step}")
    rows, V = shape
    n = n or 2 * beams
    keep = keep or min(beams, n)
    if not 1 <= beams <= BEAMS_MAX or rows % beams or not 1 <= n <= BEAMS_MAX or not 1 <= keep <= n:
        raise ValueError(f"{rows} rows of {beams} beams each, {n} candidates, {keep} that go on (at most {BEAMS_MAX})")
    if scores.dtype is not torch.float32 or scores.numel() != rows or not scores.is_contiguous():
        raise ValueError(f"scores: {rows} contiguous fp32 numbers, got {tuple(scores.shape)} {scores.dtype}")
    if ended is not None:
        _int32(ended, None, "ended")
    Q = rows // beams
    if out is None:
        _here(logits, scores, ended)
        pitch, next_pitch = 3 * n, keep
        a, b, c = scores.new_empty((Q, pitch), dtype=torch.int32).split_with_sizes((n, n, n), 1)
        d, e, f = scores.new_empty((3, Q, keep), dtype=torch.int32).unbind()
        a, d = a.view(torch.float32), d.view(torch.float32)
        out = BeamStep(a, b, c, d, e, f)
    else:
        _here(logits, scores, ended, *out)
        for t, m, what in zip(out, (n, n, n, keep, keep, keep), BeamStep._fields):
            if t.dtype is not (torch.float32 if what.endswith("score") else torch.int32) or t.numel() != Q * m or not t.is_contiguous():
                raise ValueError(f"{what}: {Q} x {m} contiguous numbers, got {tuple(t.shape)} {t.dtype}")
        pitch, next_pitch = n, keep
        a, b, c, d, e, f = out
    if rows == 0:
        return out
    L = lib()
    work = scores.new_empty(_select_scratch(rows, V, n, dt, _raw_device()))
    rc = L.blitz_beam_select(logits.data_ptr(), step[0], scores.data_ptr(), rows, V, beams, n, keep, None if ended is None else ended.data_ptr(),
                             0 if ended is None else ended.shape[0], work.data_ptr(), a.data_ptr(), b.data_ptr(), c.data_ptr(), d.data_ptr(), e.data_ptr(),
                             f.data_ptr(), pitch, next_pitch, dt, _stream())
    if rc:
        _check(rc, "blitz_beam_select")
    return out


def beam_fork(table: torch.Tensor, cached: torch.Tensor, parents: torch.Tensor, pool: torch.Tensor, *, page_size: int, num_pages: int,
              out: Optional[BeamFork] = None) -> BeamFork:
    """Tables of the beams that go on.  ``table`` [requests * beams, width]: pages of the parents' rows; ``cached`` [requests * beams]: tokens
    that they hold (-1: a dead row); ``parents`` [requests, children]: the beam that each child comes from (-1: none, a dead row);
    ``pool`` [requests, n]: pages that the request owns, each once, those in use among them (-1: no page).  A child has its
    parent's full pages; a partly filled one goes to the parent's first child, and the others get a fresh page and a copy (`copy_pages`);
    where all pages are full the child gets a fresh one, so that every child has room for a token.  Fresh pages are the first ones of the pool that no
    child keeps.  A child that there is no page for is a dead row, and the status word says so.  State slots of recurrent layers move alike: a
    table of one column with pages of two tokens, of which one is there."""
    rows, W, pitch = _rows_of(table, "table")
    Q, to, parents_pitch = _rows_of(parents, "parents")
    pool_rows, P, pool_pitch = _rows_of(pool, "pool")
    k = rows // Q if Q else 1
    if rows != Q * k or not 1 <= k <= BEAMS_MAX or not 1 <= to <= BEAMS_MAX or W < 1 or to * W >= 1 << 31:
        raise ValueError(f"a table of {rows} rows of {W} pages for {Q} requests with {to} children each (at most {BEAMS_MAX} beams)")
    if page_size < 1 or not 1 <= num_pages <= 1600000:
        raise ValueError(f"{num_pages} pages of {page_size} tokens")
    if pool_rows != Q:
        raise ValueError(f"pool: a row for each of {Q} requests, got {tuple(pool.shape)}")
    _numbers(cached, rows, "cached")
    if out is None:
        _here(table, cached, parents, pool)
        R = Q * to
        new, a, b, c, d = table.new_empty(R * (W + 4)).split_with_sizes((R * W, R, R, R, R))
        out = BeamFork(new.view(R, W), a, b, c, d)
    else:
        _here(table, cached, parents, pool, *out)
        _ints(out.table, (Q * to, W), "out.table")
        for t in out[1:]:
            _ints(t, (Q * to,), "out")
        if out.table.untyped_storage().data_ptr() == table.untyped_storage().data_ptr() and \
                out.table.data_ptr() < table.data_ptr() + 4 * ((rows - 1) * pitch + W) and table.data_ptr() < out.table.data_ptr() + 4 * Q * to * W:
            raise ValueError("out.table shares memory with the table")
    a, b, c, d, e = out
    rc = lib().blitz_beam_fork(table.data_ptr(), pitch, cached.data_ptr(), parents.data_ptr(), parents_pitch, pool.data_ptr(), pool_pitch, Q, k, to, W, P, page_size, num_pages,
                               a.data_ptr(), b.data_ptr(), c.data_ptr(), d.data_ptr(), e.data_ptr(), _status_ptr(table), _stream())
    if rc:
        _check(rc, "blitz_beam_fork")
    return out


def _copy(t: torch.Tensor, layers: bool, parts: int, page: int, src, dst, tokens) -> None:
    """Copies in one tensor [layers?, pages, ...]; parts > 0: pages are that many runs of `page` tokens."""
    shape, i = t.shape, 1 if layers else 0
    if not t.is_contiguous() or len(shape) < 1 + i:
        raise ValueError(f"a cache is one contiguous tensor, got {tuple(shape)}, strides {t.stride()}")
    whole, n, pages = t.stride(i) * t.element_size(), src.shape[0], shape[i]
    if n == 0 or t.numel() == 0:
        return
    run = whole // parts
    rc = lib().blitz_copy_pages(t.data_ptr(), shape[0] if layers else 1, pages * whole, pages, whole, parts, run, run, run // page, src.data_ptr(), dst.data_ptr(),
                                None if tokens is None else tokens.data_ptr(), n, _status_ptr(t), _stream())
    if rc:
        _check(rc, "blitz_copy_pages")


def copy_pages(cache: Union[torch.Tensor, KVPair, LatentKV, QuantKV], src: torch.Tensor, dst: torch.Tensor, tokens: Optional[torch.Tensor] = None, *,
               layers: bool = False) -> None:
    """Page ``src[i]`` of a cache to page ``dst[i]``; pairs with a negative number are left out.  ``layers``: a tensor whose first dimension
    is the layers, all of which are copied.  With ``tokens``, only the first tokens[i] of a page [2, page, kv_heads, dim] (or of a KVPair's or
    LatentKV's pages); without, whole pages, of a tensor of any kind: bytes of a 4-bit cache (always whole), states by slot.  A page is the
    destination of one pair at most, and of none if it is a source."""
    n = _int32(src, None, "src").shape[0]
    _int32(dst, n, "dst")
    if tokens is not None:
        _int32(tokens, n, "tokens")
    if isinstance(cache, torch.Tensor):
        _here(cache, src, dst, tokens)
        if tokens is None:
            return _copy(cache, layers, 1, 1, src, dst, None)
        if cache.dim() != 5 + layers or cache.shape[1 + layers] != 2:
            raise ValueError(f"tokens of pages [2, page, kv_heads, dim], got a cache {tuple(cache.shape)}")
        return _copy(cache, layers, 2, max(1, cache.shape[2 + layers]), src, dst, tokens)
    if layers:
        raise ValueError("layers: of one tensor")
    if isinstance(cache, QuantKV):
        _copy(_quant(cache, src, dst), False, 1, 1, src, dst, None)
    else:
        for t in cache if isinstance(cache, KVPair) else (cache.pool,):
            _here(t, src, dst, tokens)
            if t.dim() != 4:
                raise ValueError(f"pages [page, heads, dim], got {tuple(t.shape)}")
            _copy(t, False, 1, max(1, t.shape[1]), src, dst, tokens)


def step_tables(table: torch.Tensor, cached: torch.Tensor, counts: Optional[torch.Tensor] = None, *, page_size: int, beams: int = 0, tokens: int = 0,
                entries: int = 0, out: Optional[StepTables] = None) -> StepTables:
    """The tables of a step.  ``table`` [rows, width]: pages of every row, those for its new tokens among them; ``cached`` [rows]: tokens that
    it holds (-1: padding).  Without ``counts`` every row has one new token and its place in ``pos`` and ``slot`` (padding: 0 and -1), as decode steps take
    them.  With ``counts`` [rows] row r has that many, one row's behind the other's in the ``tokens`` places of pos and slot, and rows without
    new tokens have no pages.  ``entries`` (rows * width): places for pages.  Behind the last: page 0, position 0, slot -1.  ``beams`` > 0: full
    pages, new tokens counted, that the rows of each group of so many have in common.  Rows that do not fit into ``entries`` or ``tokens``, and all
    behind them, sit the step out, as does one whose tokens its table has no place for; the status word says so."""
    R, W, pitch = _rows_of(table, "table")
    _numbers(cached, R, "cached")
    entries = entries or R * W
    ragged = counts is not None
    if page_size < 1 or W < 1 or R * W * page_size >= 1 << 31 or not 0 <= R <= 8192 or entries < 0 or tokens < 0 or beams < 0 or (beams and R % beams):
        raise ValueError(f"{R} rows of {W} pages of {page_size} tokens, {beams} beams, {entries} entries, {tokens} tokens")
    if ragged:
        _numbers(counts, R, "counts")
    elif tokens:
        raise ValueError("tokens: with counts")
    T = tokens if ragged else R
    if out is None:
        _here(table, cached, counts)
        x, y = R + 1 if ragged else 0, R // beams if beams else 0
        a, b, c, d, e, f, g = table.new_empty(entries + 2 * (R + T) + 1 + x + y).split_with_sizes((entries, R + 1, R, T, T, x, y))
        out = StepTables(a, b, c, d, e, f if ragged else None, g if beams else None)
    else:
        sizes = (entries, R + 1, R, T, T, R + 1 if ragged else None, R // beams if beams else None)
        for t, n, what in zip(out, sizes, StepTables._fields):
            if (t is None) != (n is None):
                raise ValueError(f"out.{what}: {'missing' if t is None else 'not asked for'}")
            if t is not None:
                _ints(t, (n,), "out." + what)
        _here(table, cached, counts, *out)
    if R == 0:
        for t in out[:2] + out[3:6]:
            if t is not None:
                t.zero_()
        out.slot.fill_(-1)
        return out
    a, b, c, d, e, f, g = out
    rc = lib().blitz_step_tables(table.data_ptr(), pitch, cached.data_ptr(), counts.data_ptr() if ragged else None, R, W, page_size, beams, entries, tokens, a.data_ptr(),
                                 b.data_ptr(), c.data_ptr(), d.data_ptr(), e.data_ptr(), None if f is None else f.data_ptr(), None if g is None else g.data_ptr(),
                                 _status_ptr(table), _stream())
    if rc:
        _check(rc, "blitz_step_tables")
    return out


def attn_beams_workspace_bytes(rows: int, beams: int, *, q_heads: int, kv_heads: int, head_dim: int, device=None) -> int:
    """Scratch of `attn_decode_beams` for calls of up to ``rows`` rows in groups of ``beams``: for one call at a time, nothing is kept in it."""
    with torch.cuda.device(device):         # (None: the current one)
        return int(lib().blitz_attn_beams_workspace_bytes(rows, beams, q_heads, kv_heads, head_dim))


def attn_decode_beams(q: torch.Tensor, kv_layer: torch.Tensor, indices: torch.Tensor, indptr: torch.Tensor, last_page_len: torch.Tensor, shared: torch.Tensor, *,
                      beams: int, q_heads: int, kv_heads: int, head_dim: int, page_size: int, workspace: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None, softcap: float = 0.0, sink: Optional[torch.Tensor] = None,
                      static_table: bool = False) -> torch.Tensor:
    """Decode attention (see `attn_decode`) of rows in groups of ``beams`` whose first pages are the same: the first ``shared`` [rows / beams] pages
    of a group, full in every row of it that has pages, are read once for all its rows.  Scores of -inf have no weight; a row of nothing else is NaN, as its softmax (zeros with a ``sink``).  Sums are fp32: finite as long as tokens
    times the largest value is.  q [rows, >= q_heads * head_dim]; a 16-bit cache of heads of 64 or 128
    [pages, 2, page, kv_heads, dim], pages of 16 tokens times a power of two; rows without pages are zeros."""
    dt = q.dtype
    if dt not in _DT:
        raise TypeError(f"kernels take fp16/bf16 tensors, got {dt}")
    if not isinstance(kv_layer, torch.Tensor):
        raise ValueError("attention of beams reads a 16-bit cache of one tensor; other caches go through attn_decode")
    R, width, shape = _int32(indptr, 1, "indptr").shape[0] - 1, q_heads * head_dim, kv_layer.shape
    if head_dim not in (64, 128) or kv_heads < 1 or q_heads < 1 or q_heads % kv_heads or page_size < 16 or page_size & (page_size - 1):
        raise ValueError(f"{q_heads} query and {kv_heads} KV heads of {head_dim}, pages of {page_size} tokens")
    if kv_layer.dtype is not dt or shape[1:] != (2, page_size, kv_heads, head_dim) or shape[0] < 1 or not kv_layer.is_contiguous() or kv_layer.data_ptr() & 15:
        raise ValueError(f"a cache [pages, 2, {page_size}, {kv_heads}, {head_dim}] of {dt}, got {tuple(shape)} {kv_layer.dtype}")
    if not 1 <= beams <= BEAMS_MAX or R % beams:
        raise ValueError(f"{R} rows in groups of {beams} (at most {BEAMS_MAX})")
    _int32(last_page_len, R, "last_page_len")
    _int32(indices, None, "indices")
    _int32(shared, R // beams, "shared")
    if not softcap >= 0.0:
        raise ValueError(f"softcap {softcap}")
    size, step = q.shape, q.stride()
    if len(size) != 2 or size[0] < R or size[1] < width or step[1] != 1 or (step[0] | q.data_ptr() >> 1) & 7:
        raise ValueError(f"q: {R} rows of {q_heads} heads of {head_dim} that start on 16-byte boundaries, got {tuple(size)}, strides {step}")
    if sink is not None and (sink.dtype is not dt or sink.numel() != q_heads or not sink.is_contiguous()):
        raise ValueError(f"sink: {q_heads} numbers of {dt}")
    if out is None:
        out = q.new_empty((R, width))
    else:
        size, step = out.shape, out.stride()
        if len(size) != 2 or size[0] < R or size[1] < width or out.dtype is not dt or step[1] != 1 or (step[0] | out.data_ptr() >> 1) & 7:
            raise ValueError(f"out: {R} rows of {width} {dt} that start on 16-byte boundaries, got {tuple(size)} {out.dtype}")
    _here(q, kv_layer, indices, indptr, last_page_len, shared, out, sink, workspace)
    if R == 0:
        return out
    L = lib()
    if workspace is None:
        workspace = q.new_empty(_attn_scratch(R, beams, q_heads, kv_heads, head_dim, _raw_device()), dtype=torch.uint8)
    elif workspace.dtype is not torch.uint8 or not workspace.is_contiguous() or workspace.data_ptr() & 255:
        raise ValueError(f"workspace: bytes that start on a 256-byte boundary, got {workspace.dtype}")
    rc = L.blitz_attn_beams(q.data_ptr(), q.stride(0), kv_layer.data_ptr(), indices.data_ptr(), indptr.data_ptr(), last_page_len.data_ptr(), shared.data_ptr(),
                            out.data_ptr(), out.stride(0), workspace.data_ptr(), workspace.numel(), R, beams, q_heads, kv_heads, head_dim, page_size, shape[0],
                            head_dim ** -0.5 if sm_scale is None else sm_scale, softcap, None if sink is None else sink.data_ptr(), 1 if static_table else 0,
                            _status_ptr(q), _DT[dt], _stream())
    if rc:
        need = L.blitz_attn_beams_workspace_bytes(R, beams, q_heads, kv_heads, head_dim)
        if workspace.numel() < need:
            raise ValueError(f"workspace of {workspace.numel()} bytes, {need} are needed")
        _check(rc, "blitz_attn_beams")
    return out
