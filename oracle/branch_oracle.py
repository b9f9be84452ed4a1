"""Beams, forked pages and compaction restated on the host, row by row, in
Python integers and float64 (tests only)."""
from __future__ import annotations

import math

import numpy as np

OK, E_LOGITS, E_MASKED, E_LENGTH, E_BLOCKS, E_BLOCK, E_PARENT = 0, 1, 2, 16, 17, 20, 21


def select(logits, scores, offsets, keep, finished=None):
    """dsr_select_beams: (parents, tokens, scores) of each group, and status."""
    rows = len(scores)
    status, offers = [OK] * rows, []
    for b in range(rows):
        row, c = np.asarray(logits[b], np.float64), float(scores[b])
        mine = []
        ended = finished is not None and finished[b] != 0
        if math.isnan(c) or c == math.inf:
            status[b] = E_LOGITS
        elif ended:
            mine = [(c, -1)]
        elif np.isnan(row).any() or np.isposinf(row).any():
            status[b] = E_LOGITS
        elif np.isneginf(row).all():
            status[b] = E_MASKED
        else:
            top = row.max()
            rest = math.log(math.fsum(np.exp(row - top)))  # top + rest would lose it beside a type's lowest value
            mine = [((float(x) - top) - rest + c, v) for v, x in enumerate(row)]
        offers.append([(s, v) for s, v in mine if s > -math.inf])
    groups = []
    for lo, hi in zip(offsets[:-1], offsets[1:]):
        lo, hi = min(max(int(lo), 0), rows), min(max(int(hi), 0), rows)
        best = sorted(((-s, b, v) for b in range(lo, hi) for s, v in offers[b]))[:keep]
        pad = keep - len(best)
        groups.append(([b for _, b, _ in best] + [-1] * pad, [v for _, _, v in best] + [-1] * pad,
                       [-s for s, _, _ in best] + [-math.inf] * pad))
    return groups, status


def fork(lengths, parents, table, held, shared, pool, state, blocks, page):
    """dsr_fork_pages: a dict of its results, and `copies`: (from, to, tokens)."""
    table, pool, shared = np.array(table), np.array(pool), np.array(shared)
    S, width = table.shape
    size = len(pool)
    head, count = int(state[0]), int(state[1])
    if not (0 <= head < size and 0 <= count <= size):
        head = count = 0
    fine = [L >= 0 and 0 <= h <= width and L <= h * page for L, h in zip(lengths, held)]
    rows, status, copies, children, wanted, taken = [], [], [], [0] * S, 0, 0
    for p in parents:
        p, row, st, length, lost = int(p), [], OK, 0, False
        if p < -1 or p >= S:
            st = E_PARENT
        elif p >= 0 and not fine[p]:
            st = E_LENGTH
        elif p >= 0:
            full, part = divmod(int(lengths[p]), page)
            source = [int(x) for x in table[p]]
            # the first row takes over all pages
            if children[p] == 0:
                row = source[:held[p]]
            else:
                row = source[:full]
                if part:
                    wanted += 1
                    if wanted > count:
                        st = E_BLOCKS
                    else:
                        fresh = int(pool[(head + taken) % size])
                        taken += 1
                        row = row + [fresh]
                        lost = not 0 <= source[full] < blocks  # the tokens that it should have had
                        if not lost and 0 <= fresh < blocks:
                            copies.append((source[full], fresh, part))
            if st == OK:
                children[p] += 1
                length = int(lengths[p])
                if lost or any(not 0 <= x < blocks for x in row):
                    st = E_BLOCK
            else:
                row = []
        rows.append((row, length))
        status.append(st)
    before, source_status = shared.copy(), []
    for s in range(S):
        if not fine[s]:
            source_status.append(E_LENGTH)
            continue
        full, bad = int(lengths[s]) // page, False
        for c in range(int(held[s])):
            p = int(table[s, c])
            if not 0 <= p < blocks:
                bad = True
                continue
            shared[p] += children[s] - 1 if c < full else 0 if children[s] else -1
        source_status.append(E_BLOCK if bad else OK)
    room, freed = size - count + taken, [int(p) for p in np.flatnonzero((before < 0) != (shared < 0))]
    for p in freed:
        shared[p] = 0
    for i, p in enumerate(freed[:room]):
        pool[(head + count + i) % size] = p
    out = np.full((len(rows), width), -1, np.int32)
    for r, (row, _) in enumerate(rows):
        out[r, :len(row)] = row
    return dict(table=out, held=[len(row) for row, _ in rows], lengths=[n for _, n in rows], shared=shared, pool=pool,
                state=[(head + taken) % size, count - taken + min(room, len(freed))], status=status,
                source_status=source_status, copies=copies)


def compact(table, held, shared, pool, state, blocks, page, first=0):
    """dsr_compact_pages: a dict of its results, and `copies`: (from, to, tokens)."""
    table, pool = np.array(table), np.array(pool)
    R, width = table.shape
    status, used = [], set()
    for r in range(R):
        pages = [int(x) for x in table[r, :held[r]]] if 0 <= held[r] <= width else None
        status.append(E_LENGTH if pages is None else
                      E_BLOCK if any(not 0 <= p < blocks for p in pages) else OK)
        used |= {p for p in pages or () if first <= p < blocks}
    if any(status):
        return dict(table=table, shared=shared, pool=pool, state=list(state), remap=list(range(blocks)),
                    status=status, copies=[])
    limit = first + len(used)
    src = sorted(p for p in used if p >= limit)
    dst = [p for p in range(first, limit) if p not in used]
    moved = dict(zip(src, dst))
    remap = [p if p < first else moved.get(p, p) if p in used else -1 for p in range(blocks)]
    now = None
    if shared is not None:
        now = np.zeros(blocks, np.int32)
        for p in range(blocks):
            if remap[p] >= 0:
                now[remap[p]] = shared[p]
    for r in range(R):
        table[r, :held[r]] = [remap[p] for p in table[r, :held[r]]]
    free = list(range(limit, blocks))
    return dict(table=table, shared=now, pool=free + [-1] * (len(pool) - len(free)), state=[0, len(free)],
                remap=remap, status=status, copies=[(a, b, page) for a, b in moved.items()])
