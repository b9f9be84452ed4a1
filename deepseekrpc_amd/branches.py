"""Decoding with several branches a request, on the device: parallel samples of
a prompt, or the beams of a beam search, over the paged cache of ``tree``.

A branch is a row of the batch.  ``select_beams`` picks the best continuations
of each group of beams, ``fork_pages`` makes every row the continuation of a
row of the step before (pages shared, the last one copied, freed pages back to
the pool), ``tree.plan_blocks`` and ``tree.rotary`` bring the new tokens in as
ever, and ``prefix_attention`` reads what a group of rows has in common once
for all of them.  ``compact_pages`` moves the held pages to the front of the
cache.  No function and no ``launch()`` here synchronises.

A page may be held by several rows: ``shared`` (int32 ``[blocks]``, zeros at
first) counts the rows that hold it besides one.  Rows with shared pages end
in ``fork_pages`` (no row continues them), not in ``plan_blocks``.

As in ``tree``, each operator is a function and a ``Prepared`` class whose
``launch()`` issues the marshalled call again.  The entry points and their
exact rules are declared in include/dsr_branch.h.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _native as N
from .tree import (AttentionResult, _array, _attention, _device_of, _overlap, _page, _Prepared, _requests, _rows,
                   _table, _unrecorded)

E_PARENT = N.E_PARENT
_LOGITS_TYPES = {torch.bfloat16: N.BF16, torch.float16: N.F16, torch.float32: N.F32}


def _caches(a, name, caches, dev, page, blocks, upload):
    """Caches that share their strides and are written in place: fills ``a``; the
    tensors to keep and what holds their addresses."""
    caches = list(caches)
    _unrecorded(name, *caches)
    if not caches:
        if page is None or blocks is None:
            raise ValueError("without caches, page and blocks are needed")
        a.page, a.blocks = _page(page), int(blocks)
        return caches, None
    c = caches[0]
    if not isinstance(c, torch.Tensor) or c.dim() != 4 or len(caches) > 65535:
        raise ValueError("caches must be at most 65535 tensors [blocks, page, heads, dim]")
    size = c.element_size()
    for t in caches:
        _rows(t, "caches", c.dtype, dev, c.shape)
        if t.stride() != c.stride() or t.data_ptr() % 16:
            raise ValueError("caches must share their strides and be 16-byte aligned")
    a.blocks, a.page, a.heads, a.row_bytes = c.shape[0], _page(c.shape[1]), c.shape[2], c.shape[3] * size
    if page not in (None, a.page) or blocks not in (None, a.blocks):
        raise ValueError("page and blocks must be those of the caches")
    strides = [s * size if d > 1 else 16 for s, d in zip(c.stride()[:-1], c.shape[:-1])]
    if a.row_bytes % 16 or not 16 <= a.row_bytes <= 65536 or any(s % 16 for s in strides):
        raise ValueError("cache rows must be multiples of 16 bytes, 16-byte aligned")
    if a.page * a.heads * a.row_bytes > 2**31 - 1:
        raise ValueError("a page of a cache must be less than 2^31 bytes")
    a.c_block, a.c_token, a.c_head = strides
    addresses = list(dict.fromkeys(t.data_ptr() for t in caches))  # one listed twice is moved once
    if upload:
        pointers = torch.tensor(addresses, dtype=torch.int64, device=dev)
        a.caches = pointers.data_ptr()
    else:
        pointers = (ctypes.c_void_p * len(addresses))(*addresses)
        a.host_caches = ctypes.addressof(pointers)
    a.cache_count = len(addresses)
    return caches, pointers


class _Outputs:
    """Result tensors, from ``out`` or new; what was given may not overlap
    memory that the call reads, nor other results."""

    def __init__(self, out, dev, reads):
        self.given, self.dev, self.memory = dict(out or {}), dev, dict(reads)

    def __call__(self, key, shape, dtype=torch.int32, default=None, same=None):
        """``same``: the input that the result may replace."""
        t = self.given.pop(key, None)
        if t is None:
            t = torch.empty(shape, dtype=dtype, device=self.dev) if default is None else default
        else:
            if key == "table":
                _table(t, shape[0], self.dev)
                if tuple(t.shape) != tuple(shape):
                    raise ValueError(f"out['table'] must be int32 {list(shape)}")
            else:
                _array(t, f"out['{key}']", dtype, self.dev, None)
                if tuple(t.shape) != tuple(shape):
                    raise ValueError(f"out['{key}'] must be {dtype} {list(shape)}")
            in_place = same is not None and t.data_ptr() == same.data_ptr() and t.stride() == same.stride()
            for name, other in self.memory.items():
                if other is not None and not (in_place and other is same) and _overlap(t, other):
                    raise ValueError(f"out['{key}'] must not overlap {name}")
            self.memory[f"out['{key}']"] = t
        return t

    def end(self):
        if self.given:
            raise ValueError(f"unused out tensors: {sorted(self.given)}")


# ---------------------------------------------------------------------------
# Beams.


@dataclass
class BeamResult:
    parents: torch.Tensor  # int32 [groups, keep] rows that are continued, -1: none
    tokens: torch.Tensor   # int32 [groups, keep], -1: an ended row itself (or none)
    scores: torch.Tensor   # float64 [groups, keep], best first
    status: torch.Tensor   # int32 [rows]


class PreparedBeams(_Prepared):
    """See ``select_beams``."""

    def __init__(self, logits, scores, offsets, *, keep: int, finished=None, out: dict | None = None):
        dev = _device_of(logits, "logits")
        _unrecorded("select_beams", logits, scores)
        if logits.dim() != 2 or logits.dtype not in _LOGITS_TYPES:
            raise ValueError("logits must be bf16/f16/f32 of shape [rows, V]")
        rows, V = logits.shape
        if rows > N.BEAMS_MAX_ROWS or not 1 <= V <= N.BEAMS_MAX_VOCAB:
            raise ValueError(f"at most {N.BEAMS_MAX_ROWS} rows of 1 to {N.BEAMS_MAX_VOCAB} logits")
        if (V > 1 and logits.stride(1) != 1) or (rows > 1 and logits.stride(0) < V):
            raise ValueError("logits must be contiguous within rows")
        if not isinstance(keep, int) or not 1 <= keep <= N.BEAMS_MAX_KEEP:
            raise ValueError(f"keep must be 1 to {N.BEAMS_MAX_KEEP}")
        a = N.SelectBeamsArgs()
        a.logits, a.dtype, a.rows, a.vocab, a.ld = logits.data_ptr(), _LOGITS_TYPES[logits.dtype], rows, V, \
            max(logits.stride(0), V)
        a.scores = _array(scores, "scores", torch.float64, dev, rows)
        a.offsets = _array(offsets, "offsets", torch.int32, dev)
        groups = offsets.numel() - 1
        if not 0 <= groups <= N.BEAMS_MAX_ROWS:
            raise ValueError(f"offsets must have 1 to {N.BEAMS_MAX_ROWS + 1} entries")
        if finished is not None:
            a.finished = _array(finished, "finished", torch.int32, dev, rows)
        take = _Outputs(out, dev, dict(logits=logits, scores=scores, offsets=offsets, finished=finished))
        res = BeamResult(take("parents", (groups, keep)), take("tokens", (groups, keep)),
                         take("scores", (groups, keep), torch.float64), take("status", (rows,)))
        take.end()
        a.parents, a.tokens, a.out_scores = (t.data_ptr() for t in (res.parents, res.tokens, res.scores))
        a.status, a.keep, a.groups = res.status.data_ptr(), keep, groups
        self._setup("dsr_select_beams", a, dev, res, (logits, scores, offsets, finished, *vars(res).values()),
                    N.load().dsr_select_beams_workspace_bytes(ctypes.byref(a)))


def select_beams(logits, scores, offsets, *, keep: int, finished=None, out: dict | None = None) -> BeamResult:
    """The ``keep`` (at most 64) best continuations of each group of beams.

    ``logits`` (bf16, f16 or f32 ``[rows, V]``) follow the rows' last tokens,
    ``scores`` (float64 ``[rows]``) are their sums of log probabilities so far,
    -inf for a place without a beam; group ``g`` is rows ``offsets[g] ..
    offsets[g + 1]`` (int32).  A row offers each token at its score plus the
    token's log softmax; one that is ``finished`` (int32 ``[rows]``, non-zero)
    offers itself at its score, as token -1.  Equal offers go to the lowest row,
    then the lowest token.  ``parents`` of the result are rows, as ``fork_pages``
    takes them.  Logarithms, sums and their order are float64.  ``out`` may
    supply the result tensors."""
    return PreparedBeams(logits, scores, offsets, keep=keep, finished=finished, out=out).launch()


# ---------------------------------------------------------------------------
# Pages.


@dataclass
class ForkResult:
    table: torch.Tensor    # int32 [rows, pages], -1 past a row's pages
    held: torch.Tensor     # int32 [rows]
    lengths: torch.Tensor  # int32 [rows]
    shared: torch.Tensor   # int32 [blocks] rows that hold each page, besides one
    pool: torch.Tensor     # the given pool, freed pages written
    state: torch.Tensor    # int32 [2]
    status: torch.Tensor   # int32 [rows]
    source_status: torch.Tensor  # int32 [sources]


class PreparedFork(_Prepared):
    """See ``fork_pages``.  The addresses of the caches go to the device once,
    for which the constructor waits for the stream; with ``upload=False`` they go
    with every launch (one for every 128 caches) and nothing waits."""

    def __init__(self, lengths, parents, table, held, shared, pool, state, caches, *, page: int | None = None,
                 blocks: int | None = None, out: dict | None = None, upload: bool = True):
        dev = _device_of(lengths, "lengths")
        S, R = _requests(lengths.numel()), _requests(parents.numel())
        a = N.ForkArgs()
        caches, pointers = _caches(a, "fork_pages", caches, dev, page, blocks, upload)
        a.lengths = _array(lengths, "lengths", torch.int32, dev)
        a.parents = _array(parents, "parents", torch.int32, dev)
        a.held = _array(held, "held", torch.int32, dev, S)
        a.table, a.table_ld, a.width = _table(table, S, dev)
        a.shared = _array(shared, "shared", torch.int32, dev, a.blocks)
        a.pool = _array(pool, "pool", torch.int32, dev)
        a.pool_state = _array(state, "state", torch.int32, dev, 2)
        if a.blocks < 1 or a.blocks * a.page > 2**31 - 1 or a.width * a.page > 2**31 - 1:
            raise ValueError("the cache and a table row must span 1 to 2^31 - 1 tokens")
        if not 1 <= pool.numel() <= 1 << 30:
            raise ValueError("pool must have 1 to 2^30 entries")
        take = _Outputs(out, dev, dict(lengths=lengths, parents=parents, table=table, held=held, shared=shared,
                                       pool=pool, state=state))
        res = ForkResult(take("table", (R, table.shape[1])), take("held", (R,)), take("lengths", (R,)),
                         take("shared", (a.blocks,), default=shared, same=shared), pool,
                         take("state", (2,), default=state, same=state), take("status", (R,)),
                         take("source_status", (S,)))
        take.end()
        a.table_out, a.table_out_ld, _ = _table(res.table, R, dev)
        for field, t in (("held_out", res.held), ("lengths_out", res.lengths), ("shared_out", res.shared),
                         ("pool_state_out", res.state), ("status", res.status),
                         ("source_status", res.source_status)):
            setattr(a, field, t.data_ptr())
        a.sources, a.rows, a.pool_size = S, R, pool.numel()
        self._setup("dsr_fork_pages", a, dev, res,
                    (lengths, parents, table, held, shared, pool, state, pointers, *caches, *vars(res).values()),
                    N.load().dsr_fork_workspace_bytes(ctypes.byref(a)))


def fork_pages(lengths, parents, table, held, shared, pool, state, caches, *, page: int | None = None,
               blocks: int | None = None, out: dict | None = None) -> ForkResult:
    """The rows of the next step, each of them the continuation of a row of this
    one: ``parents`` (int32 ``[rows]``, -1 for an empty row) names it.

    ``lengths``, ``held`` (int32 ``[sources]``) and ``table`` (int32 ``[sources,
    pages]``) are this step's rows, as ``plan_blocks`` has them; the result's are
    new tensors, for as many rows as ``parents`` has.  Full pages are shared.
    The first row that continues a source also takes its last page over; the
    others get a page of the ``pool`` and a copy of its tokens in every one of
    ``caches`` (once in one that is listed twice).  Pages that no row holds any
    more go back to the pool.  Rows that it cannot serve are empty, with a
    status.

    ``shared`` (int32 ``[blocks]``) and ``state`` are updated in place unless
    ``out`` has others; ``out`` may supply any of the results but the pool, in
    memory of their own.  Without caches, ``page`` and ``blocks`` are given.
    Caches that require a gradient are refused, but under ``torch.no_grad()``."""
    return PreparedFork(lengths, parents, table, held, shared, pool, state, caches, page=page, blocks=blocks, out=out,
                        upload=False).launch()


@dataclass
class CompactResult:
    table: torch.Tensor   # the given table (or out's), page ids rewritten
    pool: torch.Tensor    # the free pages in ascending order, -1 behind them
    state: torch.Tensor   # int32 [2]
    shared: torch.Tensor | None
    remap: torch.Tensor   # int32 [blocks] each page's new id, -1: it is free
    status: torch.Tensor  # int32 [rows]


class PreparedCompact(_Prepared):
    """See ``compact_pages``; ``upload`` as in ``PreparedFork``."""

    def __init__(self, table, held, pool, state, caches, *, shared=None, first: int = 0, page: int | None = None,
                 blocks: int | None = None, out: dict | None = None, upload: bool = True):
        dev = _device_of(held, "held")
        R = _requests(held.numel())
        a = N.CompactArgs()
        caches, pointers = _caches(a, "compact_pages", caches, dev, page, blocks, upload)
        a.held = _array(held, "held", torch.int32, dev)
        a.table, a.table_ld, a.width = _table(table, R, dev)
        a.pool = _array(pool, "pool", torch.int32, dev)
        a.pool_state = _array(state, "state", torch.int32, dev, 2)
        if a.blocks < 1 or a.blocks * a.page > 2**31 - 1 or a.width * a.page > 2**31 - 1:
            raise ValueError("the cache and a table row must span 1 to 2^31 - 1 tokens")
        a.first = int(first)
        if not 0 <= a.first < a.blocks:
            raise ValueError("first must be a page of the cache")
        if not a.blocks - a.first <= pool.numel() <= 1 << 30:
            raise ValueError("pool must have room for every page from the first on")
        if shared is not None:
            a.shared = _array(shared, "shared", torch.int32, dev, a.blocks)
        take = _Outputs(out, dev, dict(held=held, table=table, shared=shared, pool=pool, state=state))
        res = CompactResult(take("table", tuple(table.shape), default=table, same=table),
                            take("pool", tuple(pool.shape), default=pool, same=pool),
                            take("state", (2,), default=state, same=state),
                            None if shared is None else take("shared", (a.blocks,), default=shared, same=shared),
                            take("remap", (a.blocks,)), take("status", (R,)))
        take.end()
        a.table_out, a.table_out_ld, _ = _table(res.table, R, dev)
        a.shared_out = None if shared is None else res.shared.data_ptr()
        for field, t in (("pool_out", res.pool), ("pool_state_out", res.state), ("remap", res.remap),
                         ("status", res.status)):
            setattr(a, field, t.data_ptr())
        a.rows, a.pool_size = R, pool.numel()
        self._setup("dsr_compact_pages", a, dev, res,
                    (table, held, pool, state, shared, pointers, *caches, *vars(res).values()),
                    N.load().dsr_compact_workspace_bytes(ctypes.byref(a)))


def compact_pages(table, held, pool, state, caches, *, shared=None, first: int = 0, page: int | None = None,
                  blocks: int | None = None, out: dict | None = None) -> CompactResult:
    """The pages that rows hold moved to the front of the cache, from page
    ``first`` on, in every one of ``caches``: what lies behind them is free, and
    the cache may be cut there.

    ``table`` (int32 ``[rows, pages]``) and ``held`` (int32 ``[rows]``) have to be
    every row that holds pages: any other page from ``first`` on is free
    afterwards.  ``table``, ``pool``, ``state`` and ``shared`` are rewritten in
    place unless ``out`` has others.  ``remap`` of the result tells page ids that
    are kept elsewhere their new ones.  If any row has a status nothing moves.
    Without caches, ``page`` and ``blocks`` are given.  Caches that require a
    gradient are refused, but under ``torch.no_grad()``."""
    return PreparedCompact(table, held, pool, state, caches, shared=shared, first=first, page=page, blocks=blocks,
                           out=out, upload=False).launch()


# ---------------------------------------------------------------------------
# Attention.


class PreparedPrefixAttention(_Prepared):
    """See ``prefix_attention``."""

    def __init__(self, q, k_cache, v_cache, table, offsets, kv_lengths, groups, prefix_lengths, *, visible=None,
                 scale: float | None = None, lse: bool = False, out=None):
        a = N.PrefixAttentionArgs()
        res, dev, keep = _attention(a, "prefix_attention", q, k_cache, v_cache, table, offsets, kv_lengths, visible,
                                    scale, lse, out)
        a.groups = _array(groups, "groups", torch.int32, dev)
        a.group_count = groups.numel() - 1
        if not 0 <= a.group_count <= a.requests:
            raise ValueError("groups must have an entry more than there are groups, at most one for each request")
        a.prefix_lengths = _array(prefix_lengths, "prefix_lengths", torch.int32, dev, a.group_count)
        self._setup("dsr_prefix_attention", a, dev, res, (*keep, groups, prefix_lengths),
                    N.load().dsr_prefix_attention_workspace_bytes(ctypes.byref(a)))


def prefix_attention(q, k_cache, v_cache, table, offsets, kv_lengths, groups, prefix_lengths, **kw) -> AttentionResult:
    """``tree.tree_attention`` for requests that share a prefix, whose keys and
    values are read once for all of them.

    Group ``g`` is requests ``groups[g] .. groups[g + 1]`` (int32, ascending;
    requests of no group are ones without a prefix).  The first
    ``prefix_lengths[g]`` tokens (int32 ``[groups]``) of their contexts are on the
    same pages, as ``fork_pages`` leaves full pages of a common source.  The new
    tokens lie behind the prefix.  The other arguments, the result and the
    refusal of tensors that require a gradient are those of ``tree_attention``."""
    return PreparedPrefixAttention(q, k_cache, v_cache, table, offsets, kv_lengths, groups, prefix_lengths,
                                   **kw).launch()
