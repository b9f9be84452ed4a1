"""The operators of a decoding step with several branches a request, as
measurable cases.

Parallel samples of one prompt, or the beams of a beam search, are rows of one
batch over a paged cache that share the pages of what they have in common:

  select  the best continuations of each group of beams, from their logits and
          the sums of log probabilities so far
  fork    each row continues a given row of the step before: whole pages are
          shared, the page in the middle of being filled is copied in every
          layer, and pages that no row holds any more go back to the pool
  compact the held pages moved to the front of the cache, tables, pool and
          counts rewritten
  prefix  attention of the new tokens of requests that share a long prefix,
          whose keys and values are read once for all of them

`run` computes them in plain torch operations, or, with `own`, by the
launches that a program marshals once and issues per step.
"""
import math
import random
import zlib

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
NODES = 64  # most nodes of a drafted tree: one bit each in a 64-bit mask
E_MASKED, E_BLOCKS = 2, 17


# ---------------------------------------------------------------------------
# The cases.


def listed():
    return [
        # One request's few beams over a small vocabulary: latency.
        dict(name="select_one", op="select", dtype="bf16", groups=1, beams=4, vocab=32000, keep=8, masked=0.0),
        # A batch of beam searches, twice as many candidates as beams so that
        # ended ones can be set aside; some tokens are masked.
        dict(name="select_32x4", op="select", dtype="bf16", groups=32, beams=4, vocab=129280, keep=8, masked=0.3),
        # Wide beams in float32.
        dict(name="select_64x8_f32", op="select", dtype="f32", groups=64, beams=8, vocab=129280, keep=16, masked=0.0),
        # The beams of a few requests after a step of a small model.
        dict(name="fork_beams_8x4", op="fork", dtype="bf16", sources=32, family=4, rows=32, context=400, page=16, kv=8,
             dim=128, layers=4),
        # Eight samples of each of many prompts are set up at once.
        dict(name="fork_samples_256", op="fork", dtype="bf16", sources=32, family=1, rows=256, context=1024, page=64,
             kv=8, dim=128, layers=16),
        # A small cache, half of it held.
        dict(name="compact_small", op="compact", dtype="bf16", rows=16, context=500, page=16, spread=2.0, kv=4, dim=64,
             layers=4),
        # A long-running server's cache before a part of it is given up.
        dict(name="compact_128", op="compact", dtype="bf16", rows=128, context=1024, page=64, spread=2.0, kv=8,
             dim=128, layers=8),
        # The smallest call: four beams of one short prompt.
        dict(name="prefix_one", op="prefix", dtype="bf16", groups=1, family=4, alone=0, prefix_lo=992, prefix_hi=992,
             own_lo=1, own_hi=60, new_lo=1, new_hi=1, heads=32, kv=8, dim=128, page=16, trees=False, by_head=False),
        # Eight samples of each of eight prompts, a token each.
        dict(name="prefix_8x8", op="prefix", dtype="bf16", groups=8, family=8, alone=0, prefix_lo=1500, prefix_hi=8192,
             own_lo=0, own_hi=700, new_lo=1, new_hi=1, heads=64, kv=8, dim=128, page=16, trees=False, by_head=False),
        # A long document with many questions: one prefix for the whole batch.
        dict(name="prefix_1x64", op="prefix", dtype="bf16", groups=1, family=64, alone=0, prefix_lo=32768,
             prefix_hi=32768, own_lo=1, own_hi=1024, new_lo=1, new_hi=1, heads=64, kv=8, dim=128, page=64, trees=False,
             by_head=False),
        # Drafted trees behind a shared system prompt; some requests have another.
        dict(name="prefix_trees_f16", op="prefix", dtype="f16", groups=2, family=12, alone=3, prefix_lo=4000,
             prefix_hi=6000, own_lo=16, own_hi=1500, new_lo=8, new_hi=24, heads=20, kv=5, dim=96, page=32, trees=True,
             by_head=True),
        # Chunks of questions behind a few shared documents.
        dict(name="prefix_chunks", op="prefix", dtype="bf16", groups=3, family=4, alone=1, prefix_lo=6000,
             prefix_hi=12000, own_lo=0, own_hi=200, new_lo=50, new_hi=400, heads=32, kv=4, dim=128, page=32,
             trees=False, by_head=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("select", "fork", "compact", "prefix", "prefix"))
    page = rng.choice((8, 16, 32, 64, 128))
    if op == "select":
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        beams, vocab = _log(rng, 1, 16), _log(rng, 16, 150000)
        most = 512 * 129280 * 4 // (beams * vocab * BYTES[dtype])
        return dict(op=op, dtype=dtype, groups=_log(rng, 1, max(1, min(64, most))), beams=beams, vocab=vocab,
                    keep=_log(rng, 1, 64), masked=rng.choice((0.0, 0.0, 0.5, 0.99)))
    if op == "fork":
        sources = _log(rng, 1, 128)
        return dict(op=op, dtype=rng.choice(("bf16", "f16", "f32")), sources=sources, family=_log(rng, 1, 8),
                    rows=rng.choice((sources, _log(rng, 1, 256))), context=_log(rng, 1, 800), page=page,
                    kv=rng.choice((1, 2, 4)), dim=rng.choice((64, 96, 128)),
                    layers=_log(rng, 1, 16 if page < 128 else 8))
    if op == "compact":
        return dict(op=op, dtype=rng.choice(("bf16", "f16", "f32")), rows=_log(rng, 1, 100), context=_log(rng, 1, 800),
                    page=page, spread=rng.uniform(1.0, 3.0), kv=rng.choice((1, 2, 4)), dim=rng.choice((64, 96, 128)),
                    layers=_log(rng, 1, 8))
    kv = rng.choice((1, 2, 3, 4, 8))
    group = rng.choice((1, 2, 4, 5, 7, 8, 16))
    dim = rng.choice((64, 96, 128, 128, 192, 256))
    trees = rng.random() < 0.4
    groups, family = _log(rng, 1, 16), _log(rng, 1, 32)
    hi = rng.choice((1, _log(rng, 1, NODES if trees else 256)))
    # No more multiplications or cache bytes than the largest listed case.
    rows = groups * family * hi * kv * group
    prefix = max(page, int(min(64 * 64 * 33000 * 128 / (rows * dim), 33000 * 8 * 128 / (groups * kv * dim), 40000)))
    most = max(1, int(min(64 * 64 * 8000 * 128 / (rows * dim), 32 * 8192 * 8 * 128 / (groups * family * kv * dim),
                          4000)))
    prefix, ctx = _log(rng, page, max(page, prefix)), _log(rng, 1, most)
    return dict(op=op, dtype=rng.choice(("bf16", "bf16", "f16")), groups=groups, family=family,
                alone=rng.choice((0, 0, rng.randint(1, 4))), prefix_lo=rng.randint(0, prefix), prefix_hi=prefix,
                own_lo=rng.randint(0, ctx), own_hi=ctx, new_lo=rng.randint(1, hi), new_hi=hi, heads=kv * group, kv=kv,
                dim=dim, page=page, trees=trees, by_head=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# Inputs, from the seed.


def _rand(g, lo, hi, *shape):
    """Whole numbers from lo to hi, both among them."""
    return torch.randint(lo, hi + 1, shape, generator=g, device=DEV, dtype=torch.int32)


def _normal(g, dtype, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


def _chances(case):
    """A generator that depends on the case alone, for what decides shapes."""
    return random.Random(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))


def _offsets(counts):
    return torch.cat([counts.new_zeros(1), counts.cumsum(0).to(torch.int32)])


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(_PREPARE[case["op"]](case, g), case=case, op=case["op"])
    if own:
        s["handle"] = _HANDLE[case["op"]](s)
    return s


def _prepare_select(case, g):
    G, B, V = case["groups"], case["beams"], case["vocab"]
    # Logits as a projection leaves them: a few tokens well ahead of the rest.
    logits = torch.randn(G * B, V, generator=g, device=DEV) * 2.5
    logits += 4.0 * (torch.rand(G * B, V, generator=g, device=DEV) < 20.0 / V)
    if case["masked"]:
        logits.masked_fill_(torch.rand(G * B, V, generator=g, device=DEV) < case["masked"], -math.inf)
    logits = logits.to(TYPES[case["dtype"]])
    scores = -20.0 * torch.rand(G * B, generator=g, device=DEV, dtype=torch.float64)
    chance = torch.rand(G * B, generator=g, device=DEV)
    scores = torch.where(chance < 0.05, -math.inf, scores)  # a place without a beam
    finished = ((chance > 0.9) & (B > 1)).to(torch.int32)   # a beam that has ended
    return dict(logits=logits, scores=scores, finished=finished,
                offsets=torch.arange(G + 1, device=DEV, dtype=torch.int32) * B)


def _rows_of_pages(g, lengths, family, page, blocks, width):
    """Tables of rows in families of which each shares its first pages, and how
    many rows besides one hold each page.  `lengths` on the host."""
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    shared = torch.zeros(blocks, dtype=torch.int32)
    perm = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32).cpu()
    at = 0
    for first in range(0, len(lengths), family):
        rows = range(first, min(first + family, len(lengths)))
        common = min(lengths[r] // page for r in rows) * 3 // 4
        both = perm[at:at + common]
        at += common
        shared[both.long()] = len(rows) - 1
        for r in rows:
            pages = -(-lengths[r] // page)
            table[r, :common] = both
            table[r, common:pages] = perm[at:at + pages - common]
            at += pages - common
    return table.to(DEV), shared.to(DEV), perm[at:].to(DEV)


def _pool(g, free, blocks):
    """A ring of the free pages that has gone round."""
    head = int(_rand(g, 0, blocks - 1, 1))
    pool = torch.full((blocks,), -1, device=DEV, dtype=torch.int32)
    pool[(head + torch.arange(free.numel(), device=DEV)) % blocks] = free
    return pool, torch.tensor([head, free.numel()], device=DEV, dtype=torch.int32)


def _prepare_fork(case, g):
    S, R, page = case["sources"], case["rows"], case["page"]
    r = _chances(case)
    lengths = [r.randint(0, case["context"]) for _ in range(S)]
    lengths = [lengths[i] for i in torch.randperm(S, generator=g, device=DEV).tolist()]
    width = case["context"] // page + 2
    blocks = sum(-(-n // page) for n in lengths) + R + 1
    table, shared, free = _rows_of_pages(g, lengths, case["family"], page, blocks, width)
    pool, state = _pool(g, free, blocks)
    if R == S:  # a step of beams: each row continues one of its family, some rows end
        family = torch.arange(R, device=DEV) // case["family"] * case["family"]
        parents = family + (torch.rand(R, generator=g, device=DEV) * case["family"]).long()
        parents = torch.where(torch.rand(R, generator=g, device=DEV) < 1 / 16, -1, parents.clamp(max=S - 1))
    else:       # samples: rows spread over the sources
        parents = torch.arange(R, device=DEV) * S // R
    held = (table >= 0).sum(1).to(torch.int32)
    caches = _normal(g, TYPES[case["dtype"]], 2 * case["layers"], blocks, page, case["kv"], case["dim"])
    return dict(lengths=torch.tensor(lengths, device=DEV, dtype=torch.int32), parents=parents.to(torch.int32),
                table=table, held=held, shared=shared, pool=pool, state=state, caches=caches)


def _prepare_compact(case, g):
    R, page = case["rows"], case["page"]
    r = _chances(case)
    lengths = [r.randint(0, case["context"]) for _ in range(R)]
    lengths = [lengths[i] for i in torch.randperm(R, generator=g, device=DEV).tolist()]
    blocks = max(1, int(case["spread"] * sum(-(-n // page) for n in lengths)))
    table, shared, free = _rows_of_pages(g, lengths, 4, page, blocks, case["context"] // page + 2)
    pool, state = _pool(g, free, blocks)
    held = (table >= 0).sum(1).to(torch.int32)
    caches = _normal(g, TYPES[case["dtype"]], 2 * case["layers"], blocks, page, case["kv"], case["dim"])
    return dict(table=table, held=held, shared=shared, pool=pool, state=state, caches=caches)


def _trees(g, counts, offsets):
    """Masks of ancestors and self in drafted trees: node 0 is the root, every
    other node hangs on one of the eight before it."""
    back = torch.randint(1, 9, (int(offsets[-1]),), generator=g, device=DEV).tolist()
    words, at = [], 0
    for n in counts.tolist():
        mine = []
        for i in range(n):
            mine.append((mine[max(0, i - back[at + i])] if i else 0) | 1 << i)
        words += mine
        at += n
    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], device=DEV)


def _prepare_prefix(case, g):
    G, F, page = case["groups"], case["family"], case["page"]
    H, K, D = case["heads"], case["kv"], case["dim"]
    R = G * F + case["alone"]
    r = _chances(case)
    sizes = torch.tensor([(r.randint(case["new_lo"], case["new_hi"]), r.randint(case["own_lo"], case["own_hi"]))
                          for _ in range(R)], dtype=torch.int32, device=DEV)
    new, ctx = sizes[torch.randperm(R, generator=g, device=DEV)].unbind(1)
    prefix = torch.tensor([r.randint(case["prefix_lo"], case["prefix_hi"]) // page * page for _ in range(G)],
                          dtype=torch.int32, device=DEV)
    prefix = prefix[torch.randperm(G, generator=g, device=DEV)].contiguous()
    common = torch.cat([prefix.repeat_interleave(F), prefix.new_zeros(case["alone"])])
    kv_lengths = (common + ctx + new).to(torch.int32)
    pages = (kv_lengths + page - 1) // page
    blocks = int(prefix.sum()) // page + int((pages - common // page).sum()) + 1
    perm = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
    table = torch.full((R, int(pages.max())), -1, device=DEV, dtype=torch.int32)
    at, p, shares = 0, pages.tolist(), (prefix // page).tolist()
    for i, n in enumerate(shares):
        table[i * F:(i + 1) * F, :n] = perm[at:at + n]
        at += n
    for i, n in enumerate(p):
        lo = shares[i // F] if i < G * F else 0
        table[i, lo:n] = perm[at:at + n - lo]
        at += n - lo
    offsets = _offsets(new)
    dtype = TYPES[case["dtype"]]
    shape = (blocks, K, page, D) if case["by_head"] else (blocks, page, K, D)
    k_cache, v_cache = _normal(g, dtype, *shape), _normal(g, dtype, *shape)
    if case["by_head"]:
        k_cache, v_cache = k_cache.transpose(1, 2), v_cache.transpose(1, 2)
    # Heads differ in how sharply they look.
    sharp = 0.5 + 2.5 * torch.rand(H, 1, generator=g, device=DEV)
    q = (torch.randn(int(offsets[-1]), H, D, generator=g, device=DEV) * sharp).to(dtype)
    return dict(q=q, k_cache=k_cache, v_cache=v_cache, table=table, offsets=offsets, kv_lengths=kv_lengths,
                groups=torch.arange(G + 1, device=DEV, dtype=torch.int32) * F, prefix=prefix, common=common,
                visible=_trees(g, new, offsets) if case["trees"] else None, scale=D ** -0.5)


_PREPARE = dict(select=_prepare_select, fork=_prepare_fork, compact=_prepare_compact, prefix=_prepare_prefix)


# ---------------------------------------------------------------------------
# The framework's launches, marshalled once as a serving loop keeps them.


def _handle_select(s):
    from deepseekrpc_amd import branches
    return branches.PreparedBeams(s["logits"], s["scores"], s["offsets"], keep=s["case"]["keep"],
                                  finished=s["finished"])


def _handle_fork(s):
    from deepseekrpc_amd import branches
    return branches.PreparedFork(s["lengths"], s["parents"], s["table"], s["held"], s["shared"], s["pool"], s["state"],
                                 list(s["caches"]), out=dict(shared=torch.empty_like(s["shared"]),
                                                             state=torch.empty_like(s["state"])))


def _handle_compact(s):
    from deepseekrpc_amd import branches
    out = {key: torch.empty_like(s[key]) for key in ("table", "shared", "pool", "state")}
    return branches.PreparedCompact(s["table"], s["held"], s["pool"], s["state"], list(s["caches"]),
                                    shared=s["shared"], out=out)


def _handle_prefix(s):
    from deepseekrpc_amd import branches
    return branches.PreparedPrefixAttention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["offsets"],
                                            s["kv_lengths"], s["groups"], s["prefix"], visible=s["visible"],
                                            scale=s["scale"], lse=True)


_HANDLE = dict(select=_handle_select, fork=_handle_fork, compact=_handle_compact, prefix=_handle_prefix)


# ---------------------------------------------------------------------------
# One pass.


def run(s):
    return _OWN[s["op"]](s) if own else _PLAIN[s["op"]](s)


def _own_select(s):
    r = s["handle"].launch()
    return dict(parents=r.parents, tokens=r.tokens, scores=r.scores, status=r.status)


def _own_fork(s):
    r = s["handle"].launch()
    return dict(table=r.table, held=r.held, lengths=r.lengths, shared=r.shared, pool=r.pool, state=r.state,
                status=r.status, caches=s["caches"])


def _own_compact(s):
    r = s["handle"].launch()
    return dict(table=r.table, shared=r.shared, pool=r.pool, state=r.state, remap=r.remap, status=r.status,
                caches=s["caches"])


def _own_prefix(s):
    r = s["handle"].launch()
    return dict(out=r.out, lse=r.lse, status=r.status)


_OWN = dict(select=_own_select, fork=_own_fork, compact=_own_compact, prefix=_own_prefix)


def _plain_select(s):
    c = s["case"]
    G, B, V, keep = c["groups"], c["beams"], c["vocab"], c["keep"]
    # Differences between rows decide what is kept: in 64 bits.
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    alive = top > -math.inf
    x -= torch.where(alive, top, 0.0)
    x -= torch.exp(x).sum(1, keepdim=True).log()
    x += s["scores"][:, None]
    ended = s["finished"] != 0
    x = torch.where(alive & ~ended[:, None], x, -math.inf)
    # A row's last place is the beam itself, once it has ended.
    x = torch.cat([x, torch.where(ended, s["scores"], -math.inf)[:, None]], 1).view(G, -1)
    place = torch.arange(x.shape[1], device=DEV)
    best, at = [], []
    for _ in range(keep):
        b = x.amax(1, keepdim=True)
        first = torch.where(x == b, place, x.shape[1]).amin(1, keepdim=True)
        best.append(b)
        at.append(first)
        x.scatter_(1, first, -math.inf)
    best, at = torch.cat(best, 1), torch.cat(at, 1)
    none = best == -math.inf
    parents = at // (V + 1) + s["offsets"][:-1, None]
    tokens = torch.where(at % (V + 1) == V, -1, at % (V + 1))
    return dict(parents=torch.where(none, -1, parents).to(torch.int32),
                tokens=torch.where(none, -1, tokens).to(torch.int32), scores=best,
                status=torch.where(alive[:, 0] | ended, 0, E_MASKED).to(torch.int32))


def _plain_fork(s):
    page, caches = s["case"]["page"], s["caches"]
    L, P, T, H = s["lengths"].long(), s["parents"].long(), s["table"], s["held"].long()
    (S, W), R, Z = T.shape, P.numel(), s["pool"].numel()
    blocks = s["shared"].numel()
    head, count = s["state"].long()
    row, col = torch.arange(R, device=DEV), torch.arange(W, device=DEV)
    has = P >= 0
    src = P.clamp(min=0)
    # The first row that continues a source takes over its last page.
    heir = torch.full((S + 1,), R, device=DEV).scatter_reduce(0, torch.where(has, src, S), row, "amin")[:S]
    first = has & (heir[src] == row)
    full, part = L // page, L % page
    wants = (has & ~first & (part[src] > 0)).long()
    upto = wants.cumsum(0)
    short = (wants > 0) & (upto > count)
    granted = has & ~short
    wants = torch.where(short, 0, wants)
    pages = torch.where(first, H[src], full[src] + wants)
    pages = torch.where(granted, pages, 0)
    fresh = s["pool"][(head + upto - 1) % Z]
    mine = torch.where((col == full[src][:, None]) & (wants > 0)[:, None], fresh[:, None], T[src])
    table = torch.where(col < pages[:, None], mine, -1)
    # Pages gain the rows that share them and lose the ones that went on.
    rows = torch.zeros(S + 1, device=DEV, dtype=torch.long).index_add(0, torch.where(granted, src, S),
                                                                     torch.ones_like(row))[:S, None]
    change = torch.where(col < full[:, None], rows - 1, torch.where(rows > 0, 0, -1))
    on = col < H[:, None]
    shared = s["shared"].long().index_add(0, T[on].long(), change[on])
    gone = torch.nonzero(shared < 0)[:, 0]
    shared[gone] = 0
    taken = wants.sum()
    s["pool"][(head + count + torch.arange(gone.numel(), device=DEV)) % Z] = gone.to(torch.int32)
    state = torch.stack([(head + taken) % Z, count - taken + gone.numel()])
    # The copied tokens, of every layer.
    tok = torch.arange(page, device=DEV)
    r, t = torch.nonzero((wants > 0)[:, None] & (tok < part[src][:, None]), as_tuple=True)
    caches[:, fresh[r].long(), t] = caches[:, T[src[r], full[src[r]]].long(), t]
    i32 = torch.int32
    return dict(table=table, held=pages.to(i32), lengths=torch.where(granted, L[src], 0).to(i32),
                shared=shared.to(i32), pool=s["pool"], state=state.to(i32),
                status=torch.where(short, E_BLOCKS, 0).to(i32), caches=caches)


def _plain_compact(s):
    T, blocks, caches = s["table"], s["shared"].numel(), s["caches"]
    on = torch.arange(T.shape[1], device=DEV) < s["held"][:, None]
    used = torch.zeros(blocks, device=DEV, dtype=torch.bool)
    used[T[on].long()] = True
    page, n = torch.arange(blocks, device=DEV), used.sum()
    src = torch.nonzero(used & (page >= n))[:, 0]
    dst = torch.nonzero(~used & (page < n))[:, 0]
    remap = torch.where(used, page, -1)
    remap[src] = dst
    shared = torch.where(used, s["shared"], 0)
    shared[dst] = s["shared"][src]
    shared[src] = 0
    free = page + n
    caches[:, dst] = caches[:, src]
    i32 = torch.int32
    return dict(table=torch.where(on, remap[T.long().clamp(min=0)].to(i32), T), shared=shared,
                pool=torch.where(free < blocks, free, -1).to(i32),
                state=torch.stack([torch.zeros_like(n), blocks - n]).to(i32), remap=remap.to(i32),
                status=torch.zeros(T.shape[0], device=DEV, dtype=i32), caches=caches)


def _padded(x, counts, first, width):
    """Rows first[i] .. of x [N, ...] as [I, width, ...], zeros behind counts[i]."""
    col = torch.arange(width, device=x.device)
    at = (first[:, None].long() + col).clamp(max=max(0, x.shape[0] - 1))
    ok = col < counts[:, None]
    return torch.where(ok.reshape(ok.shape + (1,) * (x.dim() - 1)), x[at], 0)


def _partial(s, q, table, begin, end, longest, sees):
    """Attention of padded rows q [I, T, H, D] to their table rows' tokens
    begin .. end - 1: weighted values, largest score and sum of weights."""
    page, K = s["case"]["page"], s["case"]["kv"]
    I, T, H, D = q.shape
    at = begin[:, None].long() + torch.arange(max(1, longest), device=DEV)
    inside = at < end[:, None]
    block = table.long().gather(1, (at // page).clamp(max=table.shape[1] - 1)).clamp(min=0)
    keep = inside[..., None, None]
    k = torch.where(keep, s["k_cache"][block, at % page], 0).float().permute(0, 2, 3, 1).contiguous()
    v = torch.where(keep, s["v_cache"][block, at % page], 0).float().permute(0, 2, 1, 3).contiguous()
    q = q.float().view(I, T, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(I, K, -1, D).contiguous()
    score = (q @ k).mul_(s["scale"]).view(I, K, H // K, T, -1)
    ok = inside[:, None] if sees is None else inside[:, None] & sees(at)
    score.masked_fill_(~ok[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    base = torch.where(top == -math.inf, 0.0, top)
    p = score.sub_(base).exp_()
    out = (p.view(I, K, -1, p.shape[-1]) @ v).view(I, K, H // K, T, D)
    rows = lambda x: x.permute(0, 3, 1, 2, 4).reshape(I, T, H, -1)  # noqa: E731
    return rows(out), rows(top), rows(p.sum(-1, keepdim=True))


def _plain_prefix(s):
    c, offsets, kv = s["case"], s["offsets"], s["kv_lengths"].long()
    G, F, N = c["groups"], c["family"], s["q"].shape[0]
    new = offsets[1:] - offsets[:-1]
    ctx = kv - new
    i = torch.arange(N, device=DEV)
    r = torch.searchsorted(offsets[1:].contiguous(), i, right=True)
    # Each request's own tokens, under its mask.
    T = c["new_hi"]
    word = None if s["visible"] is None else _padded(s["visible"], new, offsets[:-1], T)

    def sees(at):
        j = (at - ctx[:, None])[:, None]  # index among the new tokens, negative in the context
        if word is None:
            return j <= torch.arange(T, device=DEV)[:, None]
        return (j < 0) | ((word[..., None] >> j.clamp(0, NODES - 1) & 1) > 0)

    parts = _partial(s, _padded(s["q"], new, offsets[:-1], T), s["table"], s["common"], kv, c["own_hi"] + T, sees)
    o, m, z = (x[r, i - offsets[r]] for x in parts)
    # The prefixes, once for all of a group's rows; requests behind the last group have none.
    first = offsets[s["groups"].long()]
    rows = F * T
    parts = _partial(s, _padded(s["q"], first[1:] - first[:-1], first[:-1], rows), s["table"][s["groups"][:-1].long()],
                     torch.zeros_like(s["prefix"]), s["prefix"], c["prefix_hi"], None)
    g = (r // F).clamp(max=G - 1)
    at = (i - first[g]).clamp(max=rows - 1)
    o2, m2, z2 = (x[g, at] for x in parts)
    m2 = torch.where((r < G * F)[:, None, None], m2, -math.inf)
    top = torch.maximum(m, m2)
    base = torch.where(top == -math.inf, 0.0, top)
    f, f2 = torch.exp(m - base), torch.exp(m2 - base)
    total = z * f + z2 * f2
    out = (o * f + o2 * f2) / torch.where(total == 0, 1.0, total)
    return dict(out=out.to(s["q"].dtype), lse=(top + total.log())[..., 0],
                status=torch.zeros(kv.numel(), device=DEV, dtype=torch.int32))


_PLAIN = dict(select=_plain_select, fork=_plain_fork, compact=_plain_compact, prefix=_plain_prefix)


# ---------------------------------------------------------------------------
# The definitions in 64 bits, row by row and page by page.


def exact(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = _PREPARE[case["op"]](case, g)
    return _EXACT[case["op"]](case, s)


def _exact_select(case, s):
    B, keep = case["beams"], case["keep"]
    scores = torch.full((case["groups"], keep), -math.inf, device=DEV, dtype=torch.float64)
    for i in range(case["groups"]):
        some = []
        for r in range(i * B, (i + 1) * B):
            if s["finished"][r]:
                some.append(s["scores"][r:r + 1])
                continue
            row = s["logits"][r].double()
            if float(row.max()) > -math.inf:
                some.append((row - torch.logsumexp(row, 0)).topk(min(keep, row.numel())).values + s["scores"][r])
        best = torch.cat(some).sort(descending=True).values[:keep] if some else scores[i, :0]
        scores[i, :best.numel()] = best
    return dict(parents=None, tokens=None, scores=scores, status=None)


def _exact_fork(case, s):
    page, caches = case["page"], s["caches"].double()
    L, P, T = (s[k].tolist() for k in ("lengths", "parents", "table"))
    head, count = s["state"].tolist()
    pool, known, src, dst = s["pool"].tolist(), set(), [], []
    for p in P:
        if p >= 0 and p in known and L[p] % page:
            if len(dst) == count:
                break
            src.append(T[p][L[p] // page])
            dst.append((pool[(head + len(dst)) % len(pool)], L[p] % page))
        known.add(p)
    for a, (b, n) in zip(src, dst):
        caches[:, b, :n] = caches[:, a, :n]
    none = dict.fromkeys(("table", "held", "lengths", "shared", "pool", "state", "status"))
    return dict(none, caches=caches)


def _exact_compact(case, s):
    caches = s["caches"].double()
    used = sorted({p for row, n in zip(s["table"].tolist(), s["held"].tolist()) for p in row[:n]})
    held = set(used)
    free = (p for p in range(len(used)) if p not in held)
    for p in used:
        if p >= len(used):
            caches[:, next(free)] = caches[:, p]
    none = dict.fromkeys(("table", "shared", "pool", "state", "remap", "status"))
    return dict(none, caches=caches)


def _exact_prefix(case, s):
    H, K, page = case["heads"], case["kv"], case["page"]
    out = torch.zeros(s["q"].shape, device=DEV, dtype=torch.float64)
    lse = torch.zeros(s["q"].shape[:2], device=DEV, dtype=torch.float64)
    off, kvs, table = s["offsets"].tolist(), s["kv_lengths"].tolist(), s["table"].long()
    for r, kv in enumerate(kvs):  # each request by itself, over its own table row
        lo, hi = off[r], off[r + 1]
        at = torch.arange(kv, device=DEV)
        k = s["k_cache"][table[r, at // page], at % page].double()
        v = s["v_cache"][table[r, at // page], at % page].double()
        j = at - (kv - (hi - lo))
        if s["visible"] is None:
            hidden = j[None] > torch.arange(hi - lo, device=DEV)[:, None]
        else:
            hidden = (j[None] >= 0) & ((s["visible"][lo:hi, None] >> j.clamp(min=0)[None]) % 2 == 0)
        for h in range(K):
            rows = slice(h * (H // K), (h + 1) * (H // K))
            q = s["q"][lo:hi, rows].double()
            x = torch.einsum("tgd,sd->tgs", q, k[:, h]) * s["scale"]
            x = x.masked_fill(hidden[:, None], -math.inf)
            z = torch.logsumexp(x, -1)
            lse[lo:hi, rows] = z
            out[lo:hi, rows] = torch.einsum("tgs,sd->tgd", torch.exp(x - z[..., None]), v[:, h])
    return dict(out=out, lse=lse, status=None)


_EXACT = dict(select=_exact_select, fork=_exact_fork, compact=_exact_compact, prefix=_exact_prefix)


# ---------------------------------------------------------------------------
# What one pass cannot do without.


def work(case):
    if case["op"] == "select":
        rows, V, G = case["groups"] * case["beams"], case["vocab"], case["groups"]
        # Logits; score, flag and status of a row; parents, tokens and scores.
        return dict(bytes=rows * (V * BYTES[case["dtype"]] + 16) + 16 * G * case["keep"] + 4 * (G + 1),
                    flops=3 * rows * V)
    if case["op"] == "prefix":
        e, H, K, D = BYTES[case["dtype"]], case["heads"], case["kv"], case["dim"]
        G, R = case["groups"], case["groups"] * case["family"] + case["alone"]
        new, ctx = (case["new_lo"] + case["new_hi"]) / 2, (case["own_lo"] + case["own_hi"]) / 2
        prefix = (case["prefix_lo"] + case["prefix_hi"]) / 2
        tokens = G * prefix + R * (ctx + new)  # of the cache, each read once
        rows = new * H
        return dict(bytes=tokens * (2 * K * D * e + 4 / case["page"]) + R * rows * (2 * D * e + 4) + R * 16,
                    flops=4 * D * rows * (G * case["family"] * prefix + R * (ctx + (4 if case["trees"] else new / 2))))
    # Whole numbers are few; the rows of the cache that move are the work.
    row = 2 * case["layers"] * case["kv"] * case["dim"] * BYTES[case["dtype"]]
    page, mean = case["page"], case["context"] / 2
    if case["op"] == "fork":
        S, R = case["sources"], case["rows"]
        # Of n rows that draw their parents from n, about 1 / e more draw one that is drawn already.
        copies = R * 0.37 if R == S and case["family"] > 1 else max(0, R - S) if R != S else 0
        tokens = copies * min(page - 1, mean) / 2
        return dict(bytes=2 * tokens * row + (S + R) * (mean / page * 4 + 12), flops=0)
    pages = case["rows"] * (mean / page + 0.5)
    moved = pages * (1 - 1 / case["spread"])  # the held pages that lie behind as many
    return dict(bytes=2 * moved * page * row + 8 * pages * (1 + case["spread"]), flops=0)
