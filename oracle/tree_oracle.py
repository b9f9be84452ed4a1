"""A tree-speculative decoding step restated on the host, token by token, in
Python integers and float64 (tests only)."""
from __future__ import annotations

import math

import numpy as np

OK, E_TOKEN, E_LENGTH, E_BLOCKS, E_CAPACITY, E_TREE, E_BLOCK = 0, 9, 16, 17, 18, 19, 20
MAX_NODES = 64


def is_tree(parents):
    return len(parents) <= MAX_NODES and all(-1 <= p < i for i, p in enumerate(parents))


def ancestors(parents, i):
    """Node i's path to its root: i first."""
    out = [i]
    while parents[out[-1]] >= 0:
        out.append(parents[out[-1]])
    return out


def plan(lengths, added, table, held, pool, state, blocks, page, capacity, parents=None):
    """dsr_plan_blocks, request by request.  Returns a dict of NumPy arrays
    (``table`` and ``pool`` are updated copies)."""
    table, pool = np.array(table), np.array(pool)
    R, width = table.shape
    size = len(pool)
    head, count = int(state[0]), int(state[1])
    if not (0 <= head < size and 0 <= count <= size):
        head = count = 0
    old_pool, old_table = pool.copy(), table.copy()
    wanted = returned = taken = given = tokens = 0
    off, kv, held_out, status = [0], [], [], []
    slots, positions, owners, visible = ([d] * capacity for d in (-1, 0, -1, 0))
    for r in range(R):
        L, A, h = int(lengths[r]), int(added[r]), int(held[r])
        st, bad_page = OK, False
        if L < 0 or A < -1 or h < 0 or h > width or L > h * page or L + A > width * page:
            st = E_LENGTH
        lo = min(tokens, capacity)
        tokens += max(A, 0)
        hi = min(tokens, capacity)
        off.append(hi)
        if st == OK and A > 0 and tokens > capacity:
            st = E_CAPACITY
        new_held, first = h, 0
        if st == OK and A == -1:
            returned += h
            if h > 0 and returned > size - count:
                st = E_BLOCKS
            else:
                for b in range(h):
                    pool[(head + count + returned - h + b) % size] = old_table[r, b]
                given += h
                new_held = 0
        elif st == OK:
            need = max(0, -(-(L + A) // page) - h)
            first = wanted
            wanted += need
            if need and wanted > count:
                st = E_BLOCKS
            else:
                for b in range(need):
                    table[r, h + b] = old_pool[(head + first + b) % size]
                taken += need
                new_held = h + need
        serves = st == OK and A >= 0
        tree = None
        if serves and parents is not None:
            tree = [int(p) for p in parents[lo:hi]]
            if not is_tree(tree):
                st, serves = E_TREE, False
        for i in range(lo, hi):
            owners[i] = r
            if not serves:
                continue
            j = i - lo
            b = int(table[r, (L + j) // page])
            if not 0 <= b < blocks:
                bad_page = True
                continue
            slots[i] = b * page + (L + j) % page
            path = ancestors(tree, j) if tree is not None else [0] * (j + 1)
            positions[i] = L + len(path) - 1
            if tree is not None:
                visible[i] = sum(1 << p for p in path)
        if bad_page:  # a refused request's tokens have no slot, on whatever page they would lie
            st, serves = E_BLOCK, False
            for i in range(lo, hi):
                slots[i], positions[i], visible[i] = -1, 0, 0
        kv.append(L + A if serves else 0)
        held_out.append(new_held)
        status.append(st)
    i32 = lambda x: np.asarray(x, np.int64).astype(np.int32)  # noqa: E731
    return dict(table=table, pool=pool, held=i32(held_out), state=i32([(head + taken) % size, count - taken + given]),
                offsets=i32(off), kv_lengths=i32(kv), slots=i32(slots), positions=i32(positions), owners=i32(owners),
                visible=np.array(visible, np.uint64).view(np.int64) if parents is not None else None,
                status=i32(status))


def rotate(x, positions, freqs, start, interleaved, inverse, magnitude):
    """x float64 [tokens, heads, dim], rotated."""
    x = np.array(x, np.float64)
    half = len(freqs)
    for n, p in enumerate(positions):
        for i, f in enumerate(freqs):
            a, b = (start + 2 * i, start + 2 * i + 1) if interleaved else (start + i, start + i + half)
            t = math.fmod(int(p) * float(f), 2 * math.pi) * (-1 if inverse else 1)
            c, s = math.cos(t) * magnitude, math.sin(t) * magnitude
            x[n, :, a], x[n, :, b] = x[n, :, a] * c - x[n, :, b] * s, x[n, :, a] * s + x[n, :, b] * c
    return x


def attention(q, k_cache, v_cache, table, offsets, kv_lengths, visible, scale):
    """dsr_tree_attention in float64 on arrays ``[.., heads, dim]``: out, lse,
    and sum_j p_j |v_j| (what rounding errors of the weights scale with)."""
    n, heads, dim = q.shape
    page, kv_heads = k_cache.shape[1], k_cache.shape[2]
    group = heads // kv_heads
    out, size = np.zeros((2, n, heads, dim))
    lse = np.full((n, heads), -np.inf)
    for r, kv in enumerate(kv_lengths):
        lo, hi = int(offsets[r]), int(offsets[r + 1])
        ctx = int(kv) - (hi - lo)
        if ctx < 0:
            continue
        at = np.arange(int(kv))
        k = k_cache[table[r, at // page], at % page].astype(np.float64)
        v = v_cache[table[r, at // page], at % page].astype(np.float64)
        for t in range(hi - lo):
            if visible is None:
                see = at <= ctx + t
            else:
                word = int(np.int64(visible[lo + t]).view(np.uint64))
                see = np.array([j < ctx or bool(word >> int(j - ctx) & 1) for j in at], bool)
            if not see.any():
                continue
            for h in range(heads):
                s = k[see, h // group] @ q[lo + t, h].astype(np.float64) * scale
                top = s.max()
                p = np.exp(s - top)
                lse[lo + t, h] = top + np.log(p.sum())
                p /= p.sum()
                out[lo + t, h] = p @ v[see, h // group]
                size[lo + t, h] = p @ np.abs(v[see, h // group])
    return out, lse, size


def commit(parents, tokens, sampled, offsets, kv_lengths, limit, eos, width, page, before=None):
    """dsr_commit_tree's decisions: a list of dicts, one per request
    (``eos``: a set of ids per request; ``before``: lengths, pending tokens and
    the plan's statuses)."""
    out = []
    for r, kv in enumerate(kv_lengths):
        lo, hi = int(offsets[r]), int(offsets[r + 1])
        par, n, kv = [int(p) for p in parents[lo:hi]], hi - lo, int(kv)
        d = dict(path=[], ids=[], pending=-1, stop=0, status=OK)
        if kv < n or kv > width * page or (limit[r] < 1 and (n > 0 or before is None)):
            d["status"] = E_LENGTH
        elif not is_tree(par):
            d["status"] = E_TREE
        elif n:
            d["path"] = [0]
            while True:
                t = int(sampled[lo + d["path"][-1]])
                if t < 0:
                    d = dict(path=[], ids=[], pending=-1, stop=0, status=E_TOKEN)
                    break
                d["ids"].append(t)
                reason = 1 if t in eos[r] else 2 if len(d["ids"]) >= limit[r] else 0
                child = [i for i in range(1, n) if par[i] == d["path"][-1] and int(tokens[lo + i]) == t]
                if not child:
                    d["pending"], d["stop"] = t, reason
                    break
                d["path"].append(child[0])
                if reason:
                    d["stop"] = reason
                    break
        d["length"] = 0 if d["status"] == E_LENGTH else kv - n + len(d["path"])
        if before is not None:
            length, pending, planned = (int(x[r]) for x in before)
            if planned != OK or d["status"] != OK:
                d = dict(path=[], ids=[], pending=pending, stop=0, length=length, status=planned or d["status"])
            elif n == 0:
                d["pending"] = pending
        out.append(d)
    return out
