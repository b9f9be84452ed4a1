"""The operators of a tree-speculative decoding step, as measurable cases.

A step of a target model over a paged cache, whose requests bring new tokens
(a prompt's, one decoded token, or a tree of drafted tokens):

  plan       block tables, slot maps, positions and tree masks from the
             requests' lengths, with pages taken from and given back to a pool
  rotary     rotary positions applied to queries and keys, keys and values
             written to their cache slots; or the inverse rotation alone
  attention  attention of the new tokens over the paged cache and, by causal
             order or tree mask, over each other
  commit     the accepted path of each drafted tree, and its cache rows moved
             together in every layer

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
E_LENGTH, E_BLOCKS, E_CAPACITY, E_TREE = 16, 17, 18, 19


# ---------------------------------------------------------------------------
# The cases.


def listed():
    return [
        # One decode step of a serving batch: a token per request.
        dict(name="plan_decode_64", op="plan", requests=64, new_lo=1, new_hi=1, context=16384, page=16, trees=False),
        # A tree-speculative step of a large batch.
        dict(name="plan_tree_256", op="plan", requests=256, new_lo=9, new_hi=33, context=8192, page=32, trees=True),
        # Prompt ingestion: ragged prompts, many of them continued.
        dict(name="plan_prompts_1024", op="plan", requests=1024, new_lo=0, new_hi=1023, context=2048, page=16,
             trees=False),
        # One decode step of one layer: 64 tokens into the cache.
        dict(name="rotary_decode_64", op="rotary", dtype="bf16", tokens=64, heads=64, kv=8, dim=128, rot=128, start=0,
             interleaved=False, inverse=False, scaled=False, cache=True, page=16, longest=16384),
        # A prompt chunk with interleaved pairs in the last half of the head
        # and frequencies scaled for a long context.
        dict(name="rotary_prompt_8192", op="rotary", dtype="bf16", tokens=8192, heads=64, kv=8, dim=128, rot=64,
             start=64, interleaved=True, inverse=False, scaled=True, cache=True, page=64, longest=1 << 20),
        # The gradient of a training batch's queries and keys, float32, odd sizes.
        dict(name="rotary_back_f32_2047", op="rotary", dtype="f32", tokens=2047, heads=20, kv=5, dim=80, rot=32,
             start=0, interleaved=False, inverse=True, scaled=False, cache=False, page=16, longest=8192),
        # The smallest call: one request, one token, a short context.
        dict(name="attention_one", op="attention", dtype="bf16", requests=1, new_lo=1, new_hi=1, heads=32, kv=8,
             dim=128, ctx_lo=1000, ctx_hi=1000, page=16, trees=False, by_head=False),
        # Decode of a serving batch with ragged contexts.
        dict(name="attention_decode_64", op="attention", dtype="bf16", requests=64, new_lo=1, new_hi=1, heads=64, kv=8,
             dim=128, ctx_lo=512, ctx_hi=16384, page=16, trees=False, by_head=False),
        # The usual speculative step: small drafted trees, ragged contexts.
        dict(name="attention_tree_32", op="attention", dtype="bf16", requests=32, new_lo=8, new_hi=24, heads=64, kv=8,
             dim=128, ctx_lo=256, ctx_hi=8192, page=32, trees=True, by_head=False),
        # The largest trees over long contexts, pages laid out by head.
        dict(name="attention_tree_8x64", op="attention", dtype="bf16", requests=8, new_lo=64, new_hi=64, heads=64,
             kv=8, dim=128, ctx_lo=32001, ctx_hi=32001, page=64, trees=True, by_head=True),
        # Acceptance in a small batch over the caches of a few layers.
        dict(name="commit_8", op="commit", dtype="bf16", requests=8, new_lo=16, new_hi=16, kv=8, dim=128, layers=4,
             page=16, context=200),
        # Acceptance in a full batch over the caches of a deep model.
        dict(name="commit_64", op="commit", dtype="bf16", requests=64, new_lo=17, new_hi=64, kv=8, dim=128, layers=48,
             page=16, context=200),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("plan", "rotary", "attention", "attention", "commit"))
    page = rng.choice((1, 8, 16, 32, 64, 128))
    if op == "plan":
        requests, trees = _log(rng, 1, 1024), rng.random() < 0.5
        hi = _log(rng, 1, NODES if trees else 1023)
        return dict(op=op, requests=requests, new_lo=rng.randint(0, hi), new_hi=hi, context=_log(rng, 1, 16384),
                    page=max(page, 8), trees=trees)
    if op == "rotary":
        kv = rng.randint(1, 8)
        dim = rng.choice((64, 80, 96, 128, 192, 256))
        heads = kv * rng.randint(1, 8)
        rot = rng.choice((dim, dim // 2, 32, 24))
        inverse = rng.random() < 0.25
        most = 8192 * 72 * 128 // ((heads + 2 * kv) * dim)
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        return dict(op=op, dtype=dtype, tokens=_log(rng, 1, min(8192, most if dtype != "f32" else most // 2)),
                    heads=heads, kv=kv, dim=dim, rot=rot, start=rng.choice((0, dim - rot)),
                    interleaved=rng.random() < 0.5, inverse=inverse, scaled=rng.random() < 0.5, cache=not inverse,
                    page=page, longest=_log(rng, 2, 1 << 20))
    if op == "attention":
        kv = rng.choice((1, 2, 3, 4, 8))
        group = rng.choice((1, 2, 4, 5, 7, 8, 16))
        dim = rng.choice((64, 96, 128, 128, 192, 256))
        trees = rng.random() < 0.6
        hi = _log(rng, 1, NODES if trees else 512)
        lo = _log(rng, 1, hi)
        requests = _log(rng, 1, 128)
        # No more multiplications or cache bytes than the largest listed cases.
        most = min(8 * 64 * 64 * 32001 * 128 / (requests * hi * kv * group * dim),
                   64 * 8192 * 8 * 128 / (requests * kv * dim), 65536)
        ctx = _log(rng, 1, max(2, int(most)))
        return dict(op=op, dtype=rng.choice(("bf16", "bf16", "f16")), requests=requests, new_lo=lo, new_hi=hi,
                    heads=kv * group, kv=kv, dim=dim, ctx_lo=rng.randint(0, ctx), ctx_hi=ctx, page=page, trees=trees,
                    by_head=rng.random() < 0.5)
    hi = _log(rng, 2, NODES)
    return dict(op=op, dtype=rng.choice(("bf16", "f16")), requests=_log(rng, 1, 64), new_lo=rng.randint(1, hi),
                new_hi=hi, kv=rng.choice((1, 2, 4, 8)), dim=rng.choice((64, 96, 128)), layers=_log(rng, 1, 48),
                page=page, context=rng.randint(0, 200))


# ---------------------------------------------------------------------------
# Inputs, from the seed.


def _rand(g, lo, hi, *shape):
    """Whole numbers from lo to hi, both among them."""
    return torch.randint(lo, hi + 1, shape, generator=g, device=DEV, dtype=torch.int32)


def _sizes(g, case, lo, hi, context_lo, context_hi):
    """New tokens and context of each request.  Only the case decides them,
    so that every seed's outputs have one shape; the seed orders the requests."""
    r = random.Random(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))
    pairs = [(r.randint(lo, hi), r.randint(context_lo, context_hi)) for _ in range(case["requests"])]
    pairs = torch.tensor(pairs, dtype=torch.int32, device=DEV)
    new, ctx = pairs[torch.randperm(case["requests"], generator=g, device=DEV)].unbind(1)
    return new.contiguous(), ctx.contiguous()


def _normal(g, dtype, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _offsets(counts):
    return torch.cat([counts.new_zeros(1), counts.cumsum(0).to(torch.int32)])


def _parents(g, counts):
    """Parents of drafted trees, request after request: node 0 is the root
    (parent -1), every other node hangs on one of the eight before it."""
    off = _offsets(counts).long()
    n = int(off[-1])
    owner = torch.repeat_interleave(torch.arange(counts.numel(), device=DEV), counts.long(), output_size=n)
    local = torch.arange(n, device=DEV) - off[owner]
    back = torch.randint(1, 9, (n,), generator=g, device=DEV)
    return torch.where(local == 0, -1, (local - back).clamp(min=0)).to(torch.int32)


def _table(g, pages, blocks):
    """A block table whose row r owns pages[r] different blocks, in no order;
    the entries past them are -1."""
    width = max(1, int(pages.max()))
    perm = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
    first = pages.long().cumsum(0) - pages.long()
    col = torch.arange(width, device=DEV)
    at = (first[:, None] + col).clamp(max=blocks - 1)
    return torch.where(col < pages[:, None], perm[at], -1).to(torch.int32), perm


def _frequencies(case):
    """Radians per position of each pair: base 10,000; scaled for long
    contexts, the slow pairs are stretched eight times and the ones between
    are blended (a ramp over the pairs that turn 1 to 32 times in 8,192)."""
    half = case["rot"] // 2
    f = 10000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) * 2 / case["rot"])
    if case["scaled"]:
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1) / 31).clamp(0, 1)
        f = f * keep + f / 8 * (1 - keep)
    return f


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(_PREPARE[case["op"]](case, g), case=case, op=case["op"])
    if own:
        s["handle"] = _HANDLE[case["op"]](s)
    return s


def _prepare_plan(case, g):
    R, page = case["requests"], case["page"]
    added, lengths = _sizes(g, case, case["new_lo"], case["new_hi"], 0, case["context"])
    held = (lengths + page - 1) // page
    width = -(-(case["context"] + case["new_hi"]) // page)
    # One in sixteen requests of the larger sizes has ended: its pages go back to the pool.
    added = torch.where(added.argsort(descending=True).argsort() < R // 16, -1, added).to(torch.int32)
    capacity = max(1, int(added.clamp(min=0).sum()))
    blocks = R * width + 1
    table, perm = _table(g, held, blocks)
    table = torch.cat([table, table.new_full((R, max(0, width - table.shape[1])), -1)], 1).contiguous()
    used = int(held.sum())
    pool = torch.full((blocks,), -1, device=DEV, dtype=torch.int32)
    head = int(_rand(g, 0, blocks - 1, 1))
    at = (head + torch.arange(blocks - used, device=DEV)) % blocks
    pool[at] = perm[used:]
    state = torch.tensor([head, blocks - used], device=DEV, dtype=torch.int32)
    parents = _parents(g, added.clamp(min=0)) if case["trees"] else None
    if parents is not None and parents.numel() == 0:
        parents = torch.full((1,), -1, device=DEV, dtype=torch.int32)
    return dict(lengths=lengths, added=added, held=held, table=table, pool=pool, state=state, parents=parents,
                blocks=blocks, capacity=capacity)


def _prepare_rotary(case, g):
    N, H, K, D = case["tokens"], case["heads"], case["kv"], case["dim"]
    dtype = TYPES[case["dtype"]]
    packed = _normal(g, dtype, N, (H + 2 * K) * D)  # as a projection leaves them: one row per token
    q = packed[:, :H * D].view(N, H, D)
    k = packed[:, H * D:(H + K) * D].view(N, K, D)
    v = packed[:, (H + K) * D:].view(N, K, D)
    s = dict(packed=packed, q=q, k=k, v=v, positions=_rand(g, 0, case["longest"] - 1, N),
             freqs=_frequencies(case), magnitude=1.0 + 0.1 * math.log(8.0) if case["scaled"] else 1.0,
             q_out=torch.empty(N, H, D, device=DEV, dtype=dtype), k_out=None)
    if case["cache"]:
        page = case["page"]
        blocks = -(-N // page) + 2
        s["slots"] = torch.randperm(blocks * page, generator=g, device=DEV)[:N].to(torch.int32)
        s["k_cache"] = torch.zeros(blocks, page, K, D, device=DEV, dtype=dtype)
        s["v_cache"] = torch.zeros(blocks, page, K, D, device=DEV, dtype=dtype)
    else:
        s["k_out"] = torch.empty(N, K, D, device=DEV, dtype=dtype)
    return s


def _prepare_attention(case, g):
    R, H, K, D, page = case["requests"], case["heads"], case["kv"], case["dim"], case["page"]
    dtype = TYPES[case["dtype"]]
    new, ctx = _sizes(g, case, case["new_lo"], case["new_hi"], case["ctx_lo"], case["ctx_hi"])
    kv_lengths = ctx + new
    pages = (kv_lengths + page - 1) // page
    blocks = int(pages.sum()) + 1
    table, _ = _table(g, pages, blocks)
    offsets = _offsets(new)
    N = int(offsets[-1])
    shape = (blocks, K, page, D) if case["by_head"] else (blocks, page, K, D)
    k_cache, v_cache = _normal(g, dtype, *shape), _normal(g, dtype, *shape)
    if case["by_head"]:
        k_cache, v_cache = k_cache.transpose(1, 2), v_cache.transpose(1, 2)
    # Heads differ in how sharply they look.
    sharp = 0.5 + 2.5 * torch.rand(H, 1, generator=g, device=DEV)
    q = (torch.randn(N, H, D, generator=g, device=DEV) * sharp).to(dtype)
    visible = None
    if case["trees"]:
        parents, _, _, seen = _ancestry(_parents(g, new), new, offsets)
        visible = _words(seen)[parents >= -1]
    return dict(q=q, k_cache=k_cache, v_cache=v_cache, table=table, offsets=offsets, kv_lengths=kv_lengths,
                visible=visible, scale=D ** -0.5, longest=case["new_hi"], deepest=case["ctx_hi"] + case["new_hi"])


def _prepare_commit(case, g):
    R, K, D, page = case["requests"], case["kv"], case["dim"], case["page"]
    dtype = TYPES[case["dtype"]]
    new, ctx = _sizes(g, case, case["new_lo"], case["new_hi"], 0, case["context"])
    kv_lengths = ctx + new
    pages = (kv_lengths + page - 1) // page
    blocks = int(pages.sum()) + 1
    table, _ = _table(g, pages, blocks)
    offsets = _offsets(new)
    N = int(offsets[-1])
    parents = _parents(g, new)
    # With a vocabulary of two, drafted tokens agree with the target's about
    # as often as a good draft's do.  Every other request has a stop token.
    tokens, sampled = _rand(g, 0, 1, N), _rand(g, 0, 1, N)
    caches = _normal(g, dtype, 2 * case["layers"], blocks, page, K, D)
    return dict(parents=parents, tokens=tokens, sampled=sampled, offsets=offsets, kv_lengths=kv_lengths, table=table,
                caches=caches, limit=_rand(g, 1, 64, R), eos=torch.ones(R, device=DEV, dtype=torch.int32),
                eos_offsets=torch.arange(R + 1, device=DEV) // 2)


_PREPARE = dict(plan=_prepare_plan, rotary=_prepare_rotary, attention=_prepare_attention, commit=_prepare_commit)


# ---------------------------------------------------------------------------
# The framework's launches, marshalled once as a serving loop keeps them.


def _handle_plan(s):
    from deepseekrpc_amd import tree
    return tree.PreparedPlan(s["lengths"], s["added"], s["table"], s["held"], s["pool"], s["state"],
                             blocks=s["blocks"], page=s["case"]["page"], capacity=s["capacity"],
                             parents=s["parents"], out=dict(held=torch.empty_like(s["held"]),
                                                            state=torch.empty_like(s["state"])))


def _handle_rotary(s):
    from deepseekrpc_amd import tree
    c = s["case"]
    cache = dict(v=s["v"], slots=s["slots"], k_cache=s["k_cache"], v_cache=s["v_cache"]) if c["cache"] else {}
    return tree.PreparedRotary(s["q"], s["k"], s["positions"], s["freqs"], start=c["start"],
                               interleaved=c["interleaved"], inverse=c["inverse"], magnitude=s["magnitude"],
                               q_out=s["q_out"], k_out=s["k_out"], **cache)


def _handle_attention(s):
    from deepseekrpc_amd import tree
    return tree.PreparedTreeAttention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["offsets"], s["kv_lengths"],
                                      visible=s["visible"], scale=s["scale"], lse=True)


def _handle_commit(s):
    from deepseekrpc_amd import tree
    return tree.PreparedCommit(s["parents"], s["tokens"], s["sampled"], s["offsets"], s["kv_lengths"], s["table"],
                               list(s["caches"]), output_limit=s["limit"], eos_offsets=s["eos_offsets"],
                               eos_ids=s["eos"])


_HANDLE = dict(plan=_handle_plan, rotary=_handle_rotary, attention=_handle_attention, commit=_handle_commit)


# ---------------------------------------------------------------------------
# One pass.


def run(s):
    return _OWN[s["op"]](s) if own else _PLAIN[s["op"]](s)


def _own_plan(s):
    r = s["handle"].launch()
    return dict(table=r.table, pool=r.pool, held=r.held, state=r.state, offsets=r.offsets, kv_lengths=r.kv_lengths,
                slots=r.slots, positions=r.positions, owners=r.owners, visible=r.visible, status=r.status)


def _own_rotary(s):
    r = s["handle"].launch()
    if s["case"]["cache"]:
        return dict(q=r.q, k_cache=s["k_cache"], v_cache=s["v_cache"])
    return dict(q=r.q, k=r.k)


def _own_attention(s):
    r = s["handle"].launch()
    return dict(out=r.out, lse=r.lse)


def _own_commit(s):
    r = s["handle"].launch()
    return dict(path=r.path, ids=r.ids, accepted=r.accepted, pending=r.pending, stop=r.stop, lengths=r.lengths,
                status=r.status, caches=s["caches"])


_OWN = dict(plan=_own_plan, rotary=_own_rotary, attention=_own_attention, commit=_own_commit)


def _padded(x, counts, offsets, width, fill):
    """x [N, ...], request after request, as [R, width, ...]."""
    col = torch.arange(width, device=x.device)
    at = (offsets[:-1, None].long() + col).clamp(max=max(0, x.shape[0] - 1))
    ok = col < counts[:, None]
    return torch.where(ok.reshape(ok.shape + (1,) * (x.dim() - 1)), x[at], fill)


def _ancestry(parents, counts, offsets):
    """Of trees padded to 64 nodes: parents (-2 where there is no node),
    whether each tree is well formed, depths, and which nodes each node sees
    (its ancestors and itself)."""
    p = _padded(parents, counts, offsets, NODES, -2).long()
    node = torch.arange(NODES, device=p.device)
    fine = ((p < node) & (p >= -2)).all(1)
    p = torch.where(fine[:, None], p, p.clamp(max=-1))
    seen = (node[:, None] == node) | ((p[..., None] == node) & (p[..., None] >= 0))
    seen = seen.float()
    for _ in range(6):  # paths of up to 64 edges
        seen = (seen @ seen > 0).float()
    seen = (seen > 0) & (p >= -1)[..., None]
    return p, fine, seen.sum(-1) - 1, seen


def _words(seen):
    """Truth values over 64 nodes as one 64-bit word."""
    bit = torch.ones((), dtype=torch.int64, device=seen.device) << torch.arange(NODES, device=seen.device)
    return (seen * bit).sum(-1)


def _plain_plan(s):
    L, A, held = s["lengths"].long(), s["added"].long(), s["held"].long()
    page, cap, blocks = s["case"]["page"], s["capacity"], s["blocks"]
    table, pool = s["table"], s["pool"]
    R, width = table.shape
    head, count = s["state"].long()
    size = pool.numel()
    done = A == -1
    fine = (L >= 0) & (A >= -1) & (held >= 0) & (held <= width) & (L <= held * page) & (L + A <= width * page)
    take = A.clamp(min=0)
    ends = take.cumsum(0)
    status = torch.where(fine, torch.where((take > 0) & (ends > cap), E_CAPACITY, 0), E_LENGTH)
    offsets = torch.cat([ends.new_zeros(1), ends]).clamp(max=cap)
    need = torch.where((status == 0) & ~done, (L + take + page - 1) // page - held, 0).clamp(min=0)
    upto = need.cumsum(0)
    short = (need > 0) & (upto > count)
    first = upto - need
    back = torch.where((status == 0) & done, held, 0)
    back_upto = back.cumsum(0)
    full = (back > 0) & (back_upto > size - count)
    status = torch.where(short | full, E_BLOCKS, status)
    need, back = torch.where(short, 0, need), torch.where(full, 0, back)
    col = torch.arange(width, device=DEV)
    # Pages given back join the pool behind its last entry.
    gives = col < back[:, None]
    at = (head + count + (back_upto - back)[:, None] + col) % size
    pool.copy_(torch.cat([pool, pool[:1]]).index_put((torch.where(gives, at, size),), table)[:size])
    # Pages taken come from its head.
    fresh = (col >= held[:, None]) & (col < (held + need)[:, None])
    got = pool[(head + first[:, None] + col - held[:, None]) % size]
    table.copy_(torch.where(fresh, got, table))
    state = torch.stack([(head + need.sum()) % size, count - need.sum() + back.sum()]).to(torch.int32)
    held_out = torch.where((status == 0) & done, 0, held + need).to(torch.int32)
    granted = (status == 0) & ~done
    # Tokens.
    i = torch.arange(cap, device=DEV)
    r = torch.searchsorted(offsets[1:].contiguous(), i, right=True)
    inside = i < offsets[-1]
    r = torch.where(inside, r, 0)
    j = i - offsets[r]
    visible, depth = None, j
    if s["parents"] is not None:
        # The capacity is exact here, so the counts are those of the offsets.
        _, well, deep, seen = _ancestry(s["parents"], take, offsets)
        bad = granted & ((take > NODES) | ~well)
        status = torch.where(bad, E_TREE, status)
        granted = granted & ~bad
        depth = deep[r, j.clamp(max=NODES - 1)].long()
        visible = torch.where(inside & granted[r], _words(seen)[r, j.clamp(max=NODES - 1)], 0)
    live = inside & granted[r]
    place = (L[r] + j).clamp(min=0)
    block = table[r, (place // page).clamp(max=width - 1)].long()
    slots = torch.where(live, block * page + place % page, -1).to(torch.int32)
    positions = torch.where(live, L[r] + depth, 0).to(torch.int32)
    return dict(table=table, pool=pool, held=held_out, state=state, offsets=offsets.to(torch.int32),
                kv_lengths=torch.where(granted, L + take, 0).to(torch.int32), slots=slots, positions=positions,
                owners=torch.where(inside, r, -1).to(torch.int32), visible=visible, status=status.to(torch.int32))


def _plain_rotary(s):
    c = s["case"]
    # Angles reach thousands of turns: they are reduced before 32 bits.
    angle = torch.remainder(s["positions"].double()[:, None] * s["freqs"], 2 * math.pi).float()
    cos, sin = torch.cos(angle) * s["magnitude"], torch.sin(angle) * s["magnitude"]
    if c["inverse"]:
        sin = -sin
    rotate = lambda x: _rotated(x.float(), cos[:, None], sin[:, None], c).to(x.dtype)  # noqa: E731
    s["q_out"].copy_(rotate(s["q"]))
    if not c["cache"]:
        s["k_out"].copy_(rotate(s["k"]))
        return dict(q=s["q_out"], k=s["k_out"])
    slot = s["slots"].long()
    s["k_cache"].view(-1, c["kv"], c["dim"])[slot] = rotate(s["k"])
    s["v_cache"].view(-1, c["kv"], c["dim"])[slot] = s["v"]
    return dict(q=s["q_out"], k_cache=s["k_cache"], v_cache=s["v_cache"])


def _rotated(x, cos, sin, c):
    lo, hi, half = c["start"], c["start"] + c["rot"], c["rot"] // 2
    part = x[..., lo:hi]
    if c["interleaved"]:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = part[..., :half], part[..., half:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([x[..., :lo], turned, x[..., hi:]], -1)


def _plain_attention(s):
    c = s["case"]
    R, H, K, D, page = c["requests"], c["heads"], c["kv"], c["dim"], c["page"]
    T, S, G = s["longest"], s["deepest"], H // K
    offsets, kv = s["offsets"], s["kv_lengths"].long()
    new = (offsets[1:] - offsets[:-1]).long()
    ctx = kv - new
    q = _padded(s["q"], new, offsets, T, 0).float()
    at = torch.arange(S, device=DEV)
    block = s["table"][:, (at // page).clamp(max=s["table"].shape[1] - 1)].long().clamp(min=0)
    inside = (at < kv[:, None])[..., None, None]
    k = torch.where(inside, s["k_cache"][block, at % page], 0).float().permute(0, 2, 3, 1).contiguous()
    v = torch.where(inside, s["v_cache"][block, at % page], 0).float().permute(0, 2, 1, 3).contiguous()
    q = q.view(R, T, K, G, D).permute(0, 2, 3, 1, 4).reshape(R, K, G * T, D).contiguous()
    score = (q @ k).view(R, K, G, T, S).mul_(s["scale"])
    j = at - ctx[:, None]  # index among the new tokens, negative in the context
    t = torch.arange(T, device=DEV)
    if s["visible"] is None:
        sees = j[:, None] <= t[:, None]
    else:
        word = _padded(s["visible"], new, offsets, T, 0)
        sees = (j[:, None] < 0) | ((word[..., None] >> j.clamp(0, NODES - 1)[:, None] & 1) > 0)
    sees = sees & (at < kv[:, None])[:, None]
    score.masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(R, K, G * T, S) @ v).view(R, K, G, T, D) / torch.where(total == 0, 1.0, total)
    lse = (top + total.log())[..., 0]
    out = out.permute(0, 3, 1, 2, 4).reshape(R, T, H, D)
    lse = lse.permute(0, 3, 1, 2).reshape(R, T, H)
    i = torch.arange(s["q"].shape[0], device=DEV)
    r = torch.searchsorted(offsets[1:].contiguous(), i, right=True)
    return dict(out=out[r, i - offsets[r]].to(s["q"].dtype), lse=lse[r, i - offsets[r]])


def _plain_commit(s):
    offsets, table, caches = s["offsets"], s["table"].long(), s["caches"]
    new = (offsets[1:] - offsets[:-1]).long()
    ctx = s["kv_lengths"].long() - new
    page = caches.shape[2]
    p, fine, _, seen = _ancestry(s["parents"], new, offsets)
    tokens = _padded(s["tokens"], new, offsets, NODES, -1)
    sampled = _padded(s["sampled"], new, offsets, NODES, -1)
    wanted = sampled.gather(1, p.clamp(min=0))
    hit = (p >= 0) & (tokens == wanted)
    node = torch.arange(NODES, device=DEV)
    # Of siblings with one token the first is taken.
    rival = hit[:, None, :] & (p[:, None, :] == p[:, :, None]) & (node < node[:, None])
    hit = (hit & ~rival.any(-1)) | (node == 0)
    kept = (seen & ~hit[:, None, :]).sum(-1) == 0
    kept = kept & (p >= -1) & (fine & (new <= NODES))[:, None]
    # The path, in order; then cut behind a stop token or at the limit.
    path = torch.where(kept, node, NODES).sort(1).values
    ids = torch.where(path < NODES, sampled.gather(1, path.clamp(max=NODES - 1)), -1)
    e = s["eos_offsets"]
    stops = (ids == s["eos"][0]) & (e[1:] > e[:-1])[:, None] & (path < NODES)
    cut = stops | (node + 1 >= s["limit"][:, None])
    said = (((cut.cumsum(1) - cut.long()) == 0) & (path < NODES)).sum(1)  # ids given out
    nodes = kept.sum(1)
    # A stop at an accepted draft's token keeps that draft and asks for none after it.
    accepted = torch.minimum(said + 1, nodes)
    last = (said - 1).clamp(min=0)[:, None]
    has = nodes > 0
    stop = torch.where(stops.gather(1, last)[:, 0], 1, torch.where(said >= s["limit"], 2, 0)) * has
    pending = torch.where(has & (said == nodes), ids.gather(1, last)[:, 0], -1)
    alive = node < accepted[:, None]
    path = torch.where(alive, path, -1)
    ids = torch.where(node < said[:, None], ids, -1)
    # Cache rows: path node j's row moves to the j-th place.
    r, j = torch.nonzero(alive & (path != node), as_tuple=True)
    src, dst = ctx[r] + path[r, j], ctx[r] + j
    caches[:, table[r, dst // page], dst % page] = caches[:, table[r, src // page], src % page]
    i32 = torch.int32
    return dict(path=path.to(i32), ids=ids.to(i32), accepted=accepted.to(i32), pending=pending.to(i32),
                stop=stop.to(i32), lengths=(ctx + accepted).to(i32),
                status=torch.where(fine & (new <= NODES), 0, E_TREE).to(i32), caches=caches)


_PLAIN = dict(plan=_plain_plan, rotary=_plain_rotary, attention=_plain_attention, commit=_plain_commit)


# ---------------------------------------------------------------------------
# The definitions in 64 bits, request by request and token by token.


def exact(case, seed):
    if case["op"] == "rotary":
        return _exact_rotary(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, seed)
    if case["op"] == "commit":
        return _exact_commit(case, seed)
    return None  # whole numbers


def _state(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return _PREPARE[case["op"]](case, g)


def _exact_rotary(case, seed):
    s = _state(case, seed)
    turn = torch.polar(torch.full_like(s["freqs"], s["magnitude"])[None],
                       s["positions"].double()[:, None] * s["freqs"])  # unit numbers on the circle
    if case["inverse"]:
        turn = turn.conj()

    def rotate(x):
        y = x.double().clone()
        at = case["start"] + torch.arange(case["rot"], device=DEV)
        a, b = (at[0::2], at[1::2]) if case["interleaved"] else (at[:case["rot"] // 2], at[case["rot"] // 2:])
        z = torch.complex(y[..., a], y[..., b]) * turn[:, None]
        y[..., a], y[..., b] = z.real, z.imag
        return y

    if not case["cache"]:
        return dict(q=rotate(s["q"]), k=rotate(s["k"]))
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    b, o = s["slots"].long() // case["page"], s["slots"].long() % case["page"]
    kc[b, o] = rotate(s["k"])
    vc[b, o] = s["v"].double()
    return dict(q=rotate(s["q"]), k_cache=kc, v_cache=vc)


def _exact_attention(case, seed):
    s = _state(case, seed)
    H, K, D, page = case["heads"], case["kv"], case["dim"], case["page"]
    out = torch.zeros(s["q"].shape, device=DEV, dtype=torch.float64)
    lse = torch.zeros(s["q"].shape[:2], device=DEV, dtype=torch.float64)
    off, kvs, table = s["offsets"].tolist(), s["kv_lengths"].tolist(), s["table"].long()
    for r, kv in enumerate(kvs):
        lo, hi = off[r], off[r + 1]
        at = torch.arange(kv, device=DEV)
        k = s["k_cache"][table[r, at // page], at % page].double()
        v = s["v_cache"][table[r, at // page], at % page].double()
        new = torch.arange(hi - lo, device=DEV)
        j = at - (kv - (hi - lo))
        if s["visible"] is None:
            hidden = j[None] > new[:, None]
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
    return dict(out=out, lse=lse)


def _exact_commit(case, seed):
    s = _state(case, seed)
    page, table, caches = case["page"], s["table"].tolist(), s["caches"].double()
    off, kvs, limit, eos = (s[k].tolist() for k in ("offsets", "kv_lengths", "limit", "eos_offsets"))
    parent, token, target = (s[k].tolist() for k in ("parents", "tokens", "sampled"))
    src, dst = [], []
    for r, kv in enumerate(kvs):
        lo, hi = off[r], off[r + 1]
        ends = [1] * (eos[r + 1] - eos[r])  # every stop token is 1
        path, said = [0], 0
        while True:
            said += 1
            t = target[lo + path[-1]]
            child = [i for i in range(1, hi - lo) if parent[lo + i] == path[-1] and token[lo + i] == t]
            if child:
                path.append(child[0])
            if not child or t in ends or said >= limit[r]:
                break
        for j, i in enumerate(path):
            for row, place in ((src, kv - (hi - lo) + i), (dst, kv - (hi - lo) + j)):
                row.append(table[r][place // page] * page + place % page)
    src, dst = (torch.tensor(x, device=DEV) for x in (src, dst))
    rows = caches.flatten(1, 2)
    rows[:, dst] = rows[:, src]
    none = dict.fromkeys(("path", "ids", "accepted", "pending", "stop", "lengths", "status"))
    return dict(none, caches=caches)


# ---------------------------------------------------------------------------
# What one pass cannot do without.


def work(case):
    if case["op"] == "plan":
        R, mean = case["requests"], (case["new_lo"] + case["new_hi"]) / 2 * 15 / 16
        n = R * mean
        # Per request: length, new tokens, pages held; offset, cache length,
        # pages held, status.  Per token: slot, position, owner (and parent
        # and mask).  Per page: its pool entry and its table entry.
        return dict(bytes=28 * R + (24 if case["trees"] else 12) * n + 8 * n / case["page"] + 16,
                    flops=8 * n + 16 * R)
    if case["op"] == "rotary":
        N, e = case["tokens"], BYTES[case["dtype"]]
        per = (case["heads"] + case["kv"] * (2 if case["cache"] else 1)) * case["dim"]
        return dict(bytes=N * (2 * per * e + 4 + (4 if case["cache"] else 0)) + 4 * case["rot"],
                    flops=3 * N * (case["heads"] + case["kv"]) * case["rot"])
    if case["op"] == "attention":
        R, e = case["requests"], BYTES[case["dtype"]]
        new, ctx = (case["new_lo"] + case["new_hi"]) / 2, (case["ctx_lo"] + case["ctx_hi"]) / 2
        H, K, D = case["heads"], case["kv"], case["dim"]
        rows = R * new * H
        return dict(bytes=R * (ctx + new) * (2 * K * D * e + 4 / case["page"]) + rows * (2 * D * e + 4) + R * new * 8,
                    flops=4 * rows * D * (ctx + (new / 2 if not case["trees"] else 4)))
    R, new = case["requests"], (case["new_lo"] + case["new_hi"]) / 2
    kept = min(1.4, new - 1)  # nodes accepted behind the root, about
    row = case["kv"] * case["dim"] * BYTES[case["dtype"]]
    return dict(bytes=R * (new * 12 + 2 * NODES * 4 + 32) + 2 * R * kept * row * 2 * case["layers"],
                flops=R * new * 4)
