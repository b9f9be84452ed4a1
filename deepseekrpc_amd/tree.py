"""A tree-speculative decoding step over a paged cache, on the device.

The step around the sampler: where each request's new tokens go
(``plan_blocks``), rotary positions with keys and values written to their
cache slots (``rotary``), attention of the new tokens over the cache and each
other (``tree_attention``), and, once ``batch.sample_rows`` has drawn the
target's token at every node, the accepted path with its cache rows moved
together (``commit_tree``).  No function and no ``launch()`` here synchronises:
lengths, block tables and page pool stay on the device from step to step.

Each operator is a function and a ``Prepared`` class.  The class checks and
marshals a call once; ``launch()`` issues it on the current stream,
overwriting its outputs, as a serving loop or a graph capture does.  The
entry points and their exact rules are declared in include/dsr_tree.h.

New tokens of all requests lie one after the other; request ``r`` owns tokens
``offsets[r] .. offsets[r + 1]``.  Caches are ``[blocks, page, heads, dim]``
tensors or views with contiguous rows (head-major pages: transpose the view).
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from . import _native as N
from . import batch

MAX_NODES = N.TREE_MAX_NODES
# Statuses of requests and tokens.
E_LENGTH, E_BLOCKS, E_CAPACITY, E_TREE, E_BLOCK = N.E_LENGTH, N.E_BLOCKS, N.E_CAPACITY, N.E_TREE, N.E_BLOCK
_ROTARY_TYPES = {torch.bfloat16: N.BF16, torch.float16: N.F16, torch.float32: N.F32}
_ATTENTION_TYPES = {torch.bfloat16: N.BF16, torch.float16: N.F16}


# torch's raw accessors, as batch uses them: the public ones cost microseconds a launch.
_raw_stream = batch._raw_stream or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = batch._current_device or torch.cuda.current_device


def _device_of(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a device tensor")
    return t.device


def _unrecorded(name, *tensors):
    """A gradient that would be dropped without a word is an error."""
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        raise ValueError(f"{name} is not recorded for gradients: call it under torch.no_grad() or on detached tensors")


def _array(t, name, dtype, dev, numel=None):
    """A contiguous device array; its pointer."""
    if _device_of(t, name) != dev:
        raise ValueError(f"{name} must be on {dev}")
    if t.dtype != dtype or not t.is_contiguous() or (numel is not None and t.numel() != numel):
        raise ValueError(f"{name} must be contiguous {dtype}" + ("" if numel is None else f" with {numel} elements"))
    return t.data_ptr()


def _rows(t, name, dtype, dev, shape):
    """Rows of heads: the last dimension contiguous; pointer and the other strides."""
    if _device_of(t, name) != dev:
        raise ValueError(f"{name} must be on {dev}")
    if t.dtype != dtype or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {dtype} of shape {list(shape)}, not {t.dtype} {list(t.shape)}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous within rows")
    return (t.data_ptr(), *t.stride()[:-1])


def _overlap(a, b):
    def span(t):
        first = t.data_ptr()
        return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()

    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _table(t, rows, dev):
    if _device_of(t, "table") != dev:
        raise ValueError(f"table must be on {dev}")
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != rows or t.shape[1] < 1 or \
            (t.shape[1] > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) < t.shape[1]):
        raise ValueError("table must be int32 [requests, pages], contiguous within rows")
    return t.data_ptr(), max(t.stride(0), t.shape[1]), t.shape[1]


def _page(page):
    if not isinstance(page, int) or not 1 <= page <= N.TREE_MAX_PAGE or page & (page - 1):
        raise ValueError(f"a page holds a power of two of tokens, at most {N.TREE_MAX_PAGE}")
    return page


def _requests(n):
    if n > N.TREE_MAX_REQUESTS:
        raise ValueError(f"at most {N.TREE_MAX_REQUESTS} requests")
    return n


class _Prepared:
    """A marshalled call: ``launch()`` issues it on the current stream of its
    device.  Scratch memory is kept per stream, so launches of one object on
    two streams share its outputs only."""

    def _setup(self, name, args, device, result, keep, scratch=0):
        self.args, self.result, self.device = args, result, device
        self._keep, self._name = keep, name
        self._call = getattr(N.load(), name)
        self._ref = ctypes.byref(args)
        self._scratch, self._buffers = scratch, {}
        self._index = device.index
        self._home = self._bound = _raw_stream(self._index)
        if scratch:
            self._bind(self._home)

    def _bind(self, handle):
        if self._scratch:
            # One buffer per stream, made while the stream is current.
            ws = self._buffers.get(handle)
            if ws is None:
                ws = self._buffers[handle] = torch.empty(self._scratch, dtype=torch.uint8, device=self.device)
            self.args.workspace, self.args.workspace_bytes = ws.data_ptr(), ws.numel()
        if handle != self._home:
            # Memory of the stream it was made on: not reused before this stream is done with it.
            for t in self._keep:
                if isinstance(t, torch.Tensor) and t.is_cuda:
                    t.record_stream(torch.cuda.current_stream(self.device))
        self._bound = handle

    def launch(self):
        handle = _raw_stream(self._index)
        if handle != self._bound:
            self._bind(handle)
        if _current_device() == self._index:
            rc = self._call(self._ref, handle)
        else:
            with torch.cuda.device(self.device):
                rc = self._call(self._ref, handle)
        if rc != 0:
            N.check(rc, self._name)
        return self.result


# ---------------------------------------------------------------------------
# Block tables and slot maps.


@dataclass
class PlanResult:
    table: torch.Tensor       # the given table, new entries written
    pool: torch.Tensor        # the given pool, pages given back written
    held: torch.Tensor        # int32 [requests] pages of each request afterwards
    state: torch.Tensor       # int32 [2] the pool's first free entry and their number afterwards
    offsets: torch.Tensor     # int32 [requests + 1]
    kv_lengths: torch.Tensor  # int32 [requests] cached tokens with the new ones (0: refused or ended)
    slots: torch.Tensor       # int32 [capacity], -1: none
    positions: torch.Tensor   # int32 [capacity]
    owners: torch.Tensor      # int32 [capacity] request of each token, -1 past the last
    visible: torch.Tensor | None  # int64 [capacity] masks of ancestors and self (with parents)
    status: torch.Tensor      # int32 [requests]


def page_pool(blocks: int, device="cuda", first: int = 0):
    """A pool of the pages ``first .. blocks - 1`` of a cache: ``(pool, state)``
    as ``plan_blocks`` takes them."""
    pool = torch.arange(first, blocks, dtype=torch.int32, device=device)
    return pool, torch.tensor([0, blocks - first], dtype=torch.int32, device=device)


class PreparedPlan(_Prepared):
    """See ``plan_blocks``."""

    def __init__(self, lengths, added, table, held, pool, state, *, blocks: int, page: int, capacity: int,
                 parents=None, out: dict | None = None):
        dev = _device_of(lengths, "lengths")
        R = _requests(lengths.numel())
        capacity, blocks, page = int(capacity), int(blocks), _page(page)
        if not 1 <= capacity <= 1 << 30 or blocks < 1 or blocks * page > 2**31 - 1:
            raise ValueError("capacity must be 1 .. 2^30 and the cache hold less than 2^31 tokens")
        a = N.PlanArgs()
        a.lengths = _array(lengths, "lengths", torch.int32, dev)
        a.added = _array(added, "added", torch.int32, dev, R)
        a.held_in = _array(held, "held", torch.int32, dev, R)
        a.pool = _array(pool, "pool", torch.int32, dev)
        a.pool_state_in = _array(state, "state", torch.int32, dev, 2)
        if not 1 <= pool.numel() <= 1 << 30:
            raise ValueError("pool must have 1 to 2^30 entries")
        a.table, a.table_ld, a.width = _table(table, R, dev)
        if a.width * page > 2**31 - 1:
            raise ValueError("a table row must span less than 2^31 tokens")
        if parents is not None:
            a.parents = _array(parents, "parents", torch.int32, dev, capacity)
        out = dict(out or {})
        given = [key for key, t in out.items() if t is not None]
        i32 = lambda n: torch.empty(n, dtype=torch.int32, device=dev)  # noqa: E731

        def result(key, n, default):
            t = out.pop(key, None)
            t = default() if t is None else t
            _array(t, f"out['{key}']", torch.int32, dev, n)
            return t

        res = PlanResult(table, pool, result("held", R, lambda: held), result("state", 2, lambda: state),
                         result("offsets", R + 1, lambda: i32(R + 1)), result("kv_lengths", R, lambda: i32(R)),
                         result("slots", capacity, lambda: i32(capacity)),
                         result("positions", capacity, lambda: i32(capacity)),
                         result("owners", capacity, lambda: i32(capacity)),
                         None if parents is None else torch.empty(capacity, dtype=torch.int64, device=dev),
                         result("status", R, lambda: i32(R)))
        if out:
            raise ValueError(f"unused out tensors: {sorted(out)}")
        # Results are written while inputs and other results are still read.
        memory = dict(lengths=lengths, added=added, table=table, held=held, pool=pool, state=state, parents=parents)
        for key in given:
            t = getattr(res, key)
            if key in ("held", "state") and t.data_ptr() == memory[key].data_ptr():
                continue  # in place
            for name, other in memory.items():
                if other is not None and _overlap(t, other):
                    raise ValueError(f"out['{key}'] must not overlap {name}")
            memory[f"out['{key}']"] = t
        a.requests, a.capacity, a.page, a.pool_size, a.blocks = R, capacity, page, pool.numel(), blocks
        for field, t in (("held_out", res.held), ("pool_state_out", res.state), ("offsets", res.offsets),
                         ("kv_lengths", res.kv_lengths), ("status", res.status), ("slots", res.slots),
                         ("positions", res.positions), ("owners", res.owners), ("visible", res.visible)):
            if t is not None:
                setattr(a, field, t.data_ptr())
        self._setup("dsr_plan_blocks", a, dev, res,
                    (lengths, added, table, held, pool, state, parents, *vars(res).values()),
                    N.load().dsr_plan_workspace_bytes(R))


def plan_blocks(lengths, added, table, held, pool, state, *, blocks: int, page: int, capacity: int, parents=None,
                out: dict | None = None) -> PlanResult:
    """Pages, slots, positions and tree masks of a step's new tokens.

    ``lengths``, ``added``, ``held`` (int32 ``[requests]``): cached tokens, new
    tokens (-1: the request ends and gives its pages back) and pages held.
    ``table`` (int32 ``[requests, pages]``) gets the pages taken from the ring
    ``pool`` (int32) whose first free entry and their number are ``state``
    (int32 ``[2]``).  ``capacity`` is the length of the per-token results;
    ``parents`` (int32 ``[capacity]``, the index of each node's parent among
    its request's new tokens, -1 for none) makes them trees.  ``held`` and
    ``state`` are updated in place unless ``out`` has others; ``out`` may
    supply any of the int32 results, in memory of their own.  Requests that cannot be served are
    refused with a status, and their tokens get slot -1."""
    return PreparedPlan(lengths, added, table, held, pool, state, blocks=blocks, page=page, capacity=capacity,
                        parents=parents, out=out).launch()


# ---------------------------------------------------------------------------
# Rotary positions.


def rotary_frequencies(rot_dim: int, base: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                       original: int = 4096, slow: float = 1.0, fast: float = 32.0, device="cuda"):
    """``(freqs, magnitude)`` for ``rotary``: radians per position of each pair
    (float64), and the factor of the rotated part.

    ``scaling`` stretches them for contexts ``factor`` times ``original``:
    ``"linear"`` divides every frequency; ``"base"`` raises the base, so that
    the slowest pair is stretched by ``factor`` and the fastest not at all;
    ``"ramp"`` divides the pairs that turn less than ``slow`` times within
    ``original`` positions, keeps those that turn more than ``fast`` times,
    blends between, and sets the magnitude to 1 + 0.1 ln(factor) (YaRN)."""
    if rot_dim < 2 or rot_dim % 2 or not base > 1 or not factor >= 1:
        raise ValueError("rot_dim must be even, base above 1 and factor at least 1")
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    if scaling == "base" and rot_dim > 2:
        base = base * factor ** (rot_dim / (rot_dim - 2))
    f = base ** (-i / rot_dim)
    magnitude = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "ramp":
        keep = ((original * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        magnitude = 1.0 + 0.1 * math.log(factor)
    elif scaling not in (None, "base"):
        raise ValueError("scaling must be None, 'linear', 'base' or 'ramp'")
    return f.to(device), magnitude


@dataclass
class RotaryResult:
    q: torch.Tensor | None
    k: torch.Tensor | None
    status: torch.Tensor | None  # int32 [tokens], with a cache


class PreparedRotary(_Prepared):
    """See ``rotary``."""

    def __init__(self, q, k, positions, freqs, *, v=None, start: int = 0, interleaved: bool = False,
                 inverse: bool = False, magnitude: float = 1.0, slots=None, k_cache=None, v_cache=None, q_out=None,
                 k_out=None):
        one = q if q is not None else k
        dev = _device_of(one, "q" if q is not None else "k")
        _unrecorded("rotary", q, k, v, k_cache, v_cache, q_out, k_out)
        if one.dim() != 3 or one.dtype not in _ROTARY_TYPES:
            raise ValueError("q and k must be bf16/f16/f32 of shape [tokens, heads, dim]")
        n, dim, dtype = one.shape[0], one.shape[2], one.dtype
        if not 2 <= dim <= N.ROTARY_MAX_DIM:
            raise ValueError(f"a head has 2 to {N.ROTARY_MAX_DIM} dimensions")
        a = N.RotaryArgs()
        a.dtype, a.tokens, a.head_dim, a.magnitude = _ROTARY_TYPES[dtype], n, dim, float(magnitude)
        if not 0 < a.magnitude < 1e30:
            raise ValueError("magnitude must be positive and finite")
        a.positions = _array(positions, "positions", torch.int32, dev, n)
        a.freqs = _array(freqs, "freqs", torch.float64, dev)
        a.rot_start, a.rot_dim = int(start), 2 * freqs.numel()
        if a.rot_dim < 2 or a.rot_start < 0 or a.rot_start + a.rot_dim > dim:
            raise ValueError("the rotated part must lie within the head")
        a.interleaved, a.inverse = int(bool(interleaved)), int(bool(inverse))
        if q is not None:
            a.q, a.q_token, a.q_head = _rows(q, "q", dtype, dev, q.shape)
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=dtype, device=dev)
            a.q_out, a.qo_token, a.qo_head = _rows(q_out, "q_out", dtype, dev, q.shape)
            a.q_heads = q.shape[1]
            if q_out.data_ptr() == q.data_ptr() and q_out.stride() != q.stride():
                raise ValueError("q_out may be q itself, not another view of it")
        elif q_out is not None:
            raise ValueError("q_out needs q")
        if (slots is None) != (k_cache is None and v_cache is None) or (v is None) != (v_cache is None):
            raise ValueError("a cache needs slots, and a value cache values")
        if v is not None and k is None or k is None and (k_cache is not None or k_out is not None):
            raise ValueError("values and caches need keys")
        if k is not None:
            if k.dim() != 3:
                raise ValueError("k must be [tokens, heads, dim]")
            a.k, a.k_token, a.k_head = _rows(k, "k", dtype, dev, (n, k.shape[1], dim))
            a.kv_heads = k.shape[1]
            if k_out is None and k_cache is None:
                k_out = torch.empty(k.shape, dtype=dtype, device=dev)
            if k_out is not None:
                a.k_out, a.ko_token, a.ko_head = _rows(k_out, "k_out", dtype, dev, k.shape)
                if k_out.data_ptr() == k.data_ptr() and k_out.stride() != k.stride():
                    raise ValueError("k_out may be k itself, not another view of it")
        status = None
        if slots is not None:
            a.slots = _array(slots, "slots", torch.int32, dev, n)
            status = torch.empty(n, dtype=torch.int32, device=dev)
            a.status = status.data_ptr()
            first = k_cache if k_cache is not None else v_cache
            if first.dim() != 4:
                raise ValueError("a cache must be [blocks, page, heads, dim]")
            a.blocks, a.page = first.shape[0], _page(first.shape[1])
            if a.blocks < 1 or first.shape[0] * a.page > 2**31 - 1:
                raise ValueError("a cache must hold 1 to 2^31 - 1 tokens")
            if k_cache is not None:
                a.k_cache, a.kc_block, a.kc_token, a.kc_head = _rows(k_cache, "k_cache", dtype, dev,
                                                                     (a.blocks, a.page, a.kv_heads, dim))
            if v is not None:
                if v.dim() != 3 or not 1 <= v.shape[2] <= N.ROTARY_MAX_DIM:
                    raise ValueError("v must be [tokens, heads, dim]")
                a.v_dim = v.shape[2]
                a.v, a.v_token, a.v_head = _rows(v, "v", dtype, dev, (n, a.kv_heads, a.v_dim))
                a.v_cache, a.vc_block, a.vc_token, a.vc_head = _rows(v_cache, "v_cache", dtype, dev,
                                                                     (a.blocks, a.page, a.kv_heads, a.v_dim))
        self._setup("dsr_rotary", a, dev, RotaryResult(q_out, k_out, status),
                    (q, k, v, positions, freqs, slots, k_cache, v_cache, q_out, k_out, status))


def rotary(q, k, positions, freqs, **kw) -> RotaryResult:
    """Rotary positions of ``q`` and ``k`` (``[tokens, heads, dim]``, either may
    be None): the pairs of dimensions ``start .. start + 2 len(freqs)`` turn by
    ``position * freqs[i]`` and are multiplied by ``magnitude``; the other
    dimensions are copied.  Pairs are half a part apart, or neighbours when
    ``interleaved``.  ``inverse`` turns back: the gradient of the forward
    rotation with respect to its input.

    With ``slots`` (int32 ``[tokens]``; -1: none) the rotated keys go to
    ``k_cache`` and ``v`` to ``v_cache`` there.  Results go to ``q_out`` and
    ``k_out`` (new tensors by default, ``k_out`` only without a key cache;
    ``q`` and ``k`` themselves are allowed).

    The call is not recorded for gradients, and refuses tensors that require
    one unless recording is off.  In a ``torch.autograd.Function`` of a training
    program the backward pass is ``rotary(grad, ..., inverse=True)``."""
    return PreparedRotary(q, k, positions, freqs, **kw).launch()


# ---------------------------------------------------------------------------
# Attention.


@dataclass
class AttentionResult:
    out: torch.Tensor         # [tokens, heads, dim]
    lse: torch.Tensor | None  # float32 [tokens, heads]
    status: torch.Tensor      # int32 [requests]


class PreparedTreeAttention(_Prepared):
    """See ``tree_attention``."""

    def __init__(self, q, k_cache, v_cache, table, offsets, kv_lengths, *, visible=None, scale: float | None = None,
                 lse: bool = False, out=None):
        dev = _device_of(q, "q")
        _unrecorded("tree_attention", q, k_cache, v_cache, out)
        if q.dim() != 3 or q.dtype not in _ATTENTION_TYPES:
            raise ValueError("q must be bf16/f16 of shape [tokens, heads, dim]")
        n, heads, dim = q.shape
        if _device_of(k_cache, "k_cache") != dev or k_cache.dim() != 4:
            raise ValueError(f"k_cache must be [blocks, page, heads, dim] on {dev}")
        blocks, page, kv_heads = k_cache.shape[0], _page(k_cache.shape[1]), k_cache.shape[2]
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError("query heads must be a multiple of key heads")
        if not 8 <= dim <= N.ATTENTION_MAX_DIM or dim % 8:
            raise ValueError(f"the head dimension must be a multiple of 8 up to {N.ATTENTION_MAX_DIM}")
        R = _requests(kv_lengths.numel())
        if blocks < 1 or blocks * page > 2**31 - 1 or (n + R) * heads >= 2**29:
            raise ValueError("the cache must hold 1 to 2^31 - 1 tokens, and (tokens + requests) x heads be below 2^29")
        a = N.TreeAttentionArgs()
        shape = (blocks, page, kv_heads, dim)
        a.q, a.q_token, a.q_head = _rows(q, "q", q.dtype, dev, q.shape)
        a.k_cache, a.k_block, a.k_token, a.k_head = _rows(k_cache, "k_cache", q.dtype, dev, shape)
        a.v_cache, a.v_block, a.v_token, a.v_head = _rows(v_cache, "v_cache", q.dtype, dev, shape)
        if max(a.k_block, a.k_token, a.v_block, a.v_token) > 2**31 - 1:
            raise ValueError("strides of the caches' pages and tokens must be below 2^31")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        a.out, a.out_token, a.out_head = _rows(out, "out", q.dtype, dev, q.shape)
        for t, name in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache"), (out, "out")):
            if t.data_ptr() % 16 or any(s % 8 for s, size in zip(t.stride()[:-1], t.shape[:-1]) if size > 1):
                raise ValueError(f"rows of {name} must be 16-byte aligned")
        for field in ("q_token", "q_head", "out_token", "out_head", "k_block", "k_token", "k_head", "v_block",
                      "v_token", "v_head"):  # strides of dimensions of one element are free
            setattr(a, field, getattr(a, field) // 8 * 8)
        a.kv_lengths = _array(kv_lengths, "kv_lengths", torch.int32, dev)
        a.offsets = _array(offsets, "offsets", torch.int32, dev, R + 1)
        a.table, a.table_ld, a.width = _table(table, R, dev)
        if a.width * page > 2**31 - 1:
            raise ValueError("a table row must span less than 2^31 tokens")
        if n > 0 and R == 0:
            raise ValueError("tokens need requests")
        if visible is not None:
            a.visible = _array(visible, "visible", torch.int64, dev, n)
        a.scale = dim ** -0.5 if scale is None else float(scale)
        if not math.isfinite(a.scale):
            raise ValueError("scale must be finite")
        res = AttentionResult(out, torch.empty(n, heads, dtype=torch.float32, device=dev) if lse else None,
                              torch.empty(R, dtype=torch.int32, device=dev))
        a.lse = res.lse.data_ptr() if lse else None
        a.status = res.status.data_ptr()
        a.dtype, a.q_heads, a.kv_heads, a.head_dim = _ATTENTION_TYPES[q.dtype], heads, kv_heads, dim
        a.page, a.blocks, a.requests, a.tokens = page, blocks, R, n
        self._setup("dsr_tree_attention", a, dev, res,
                    (q, k_cache, v_cache, table, offsets, kv_lengths, visible, *vars(res).values()),
                    N.load().dsr_tree_attention_workspace_bytes(ctypes.byref(a)))


def tree_attention(q, k_cache, v_cache, table, offsets, kv_lengths, **kw) -> AttentionResult:
    """Attention of the new tokens ``q`` (``[tokens, heads, dim]``, bf16 or f16)
    over their requests' cached tokens, which include themselves: the whole
    context, and of the request's new tokens those set in ``visible`` (int64
    ``[tokens]``, as ``plan_blocks`` makes it: at most 64 new tokens a request)
    or, without it, those up to itself.  ``scale`` defaults to ``dim ** -0.5``;
    ``lse`` also returns the logarithm of each row's sum.  Rows that see nothing
    give 0 and -inf, and so do those past the last request's tokens.  ``out``
    supplies the output tensor.  There is no backward pass: tensors that require
    a gradient are refused unless recording is off."""
    return PreparedTreeAttention(q, k_cache, v_cache, table, offsets, kv_lengths, **kw).launch()


# ---------------------------------------------------------------------------
# Acceptance.


@dataclass
class CommitResult:
    path: torch.Tensor      # int32 [requests, 64] kept nodes in order, -1 padded
    ids: torch.Tensor       # int32 [requests, 64] output ids, -1 padded
    accepted: torch.Tensor  # int32 [requests] kept nodes (the root among them)
    count: torch.Tensor     # int32 [requests] output ids
    pending: torch.Tensor   # int32 [requests] the next step's root token, -1: none (kept where nothing is accepted)
    stop: torch.Tensor      # int32 [requests] STOP_NONE / STOP_EOS / STOP_LENGTH
    lengths: torch.Tensor   # int32 [requests] cached tokens afterwards
    status: torch.Tensor    # int32 [requests]


class PreparedCommit(_Prepared):
    """See ``commit_tree``.  The addresses of the caches go to the device once,
    for which the constructor waits for the stream; with ``upload=False`` they go
    with every launch (0.1 us more, and a launch for every 128 caches) and
    nothing waits."""

    def __init__(self, parents, tokens, sampled, offsets, kv_lengths, table, caches, *, output_limit,
                 eos_offsets=None, eos_ids=None, page: int | None = None, blocks: int | None = None, lengths=None,
                 pending=None, plan_status=None, upload: bool = True):
        dev = _device_of(kv_lengths, "kv_lengths")
        R = _requests(kv_lengths.numel())
        n = parents.numel()
        a = N.CommitArgs()
        a.kv_lengths = _array(kv_lengths, "kv_lengths", torch.int32, dev)
        a.parents = _array(parents, "parents", torch.int32, dev)
        a.tokens_in = _array(tokens, "tokens", torch.int32, dev, n)
        a.sampled = _array(sampled, "sampled", torch.int32, dev, n)
        a.offsets = _array(offsets, "offsets", torch.int32, dev, R + 1)
        a.output_limit = _array(output_limit, "output_limit", torch.int32, dev, R)
        a.table, a.table_ld, a.width = _table(table, R, dev)
        if (eos_offsets is None) != (eos_ids is None):
            raise ValueError("EOS ids come with their offsets")
        if eos_ids is not None and eos_ids.numel() > 0:
            a.eos_off = _array(eos_offsets, "eos_offsets", torch.int64, dev, R + 1)
            a.eos_ids = _array(eos_ids, "eos_ids", torch.int32, dev)
        before = (lengths, pending, plan_status)
        if any(t is None for t in before) != all(t is None for t in before):
            raise ValueError("lengths, pending and plan_status come together")
        if lengths is not None:
            a.lengths_in = _array(lengths, "lengths", torch.int32, dev, R)
            a.pending_in = _array(pending, "pending", torch.int32, dev, R)
            a.plan_status = _array(plan_status, "plan_status", torch.int32, dev, R)
        caches = list(caches)
        pointers = None
        if caches:
            c = caches[0]
            if c.dim() != 4 or len(caches) > 65535:
                raise ValueError("caches must be at most 65535 tensors [blocks, page, heads, dim]")
            size = c.element_size()
            for t in caches:
                _rows(t, "caches", c.dtype, dev, c.shape)
                if t.stride() != c.stride() or t.data_ptr() % 16:
                    raise ValueError("caches must share their strides and be 16-byte aligned")
            a.blocks, a.page, a.heads, a.row_bytes = c.shape[0], _page(c.shape[1]), c.shape[2], c.shape[3] * size
            strides = [s * size if d > 1 else 16 for s, d in zip(c.stride()[:-1], c.shape[:-1])]
            if a.row_bytes % 16 or not 16 <= a.row_bytes <= 65536 or any(s % 16 for s in strides):
                raise ValueError("cache rows must be multiples of 16 bytes, 16-byte aligned")
            a.c_block, a.c_token, a.c_head = strides
            addresses = list(dict.fromkeys(t.data_ptr() for t in caches))  # one listed twice is moved once
            if upload:
                pointers = torch.tensor(addresses, dtype=torch.int64, device=dev)
                a.caches = pointers.data_ptr()
            else:
                pointers = (ctypes.c_void_p * len(addresses))(*addresses)
                a.host_caches = ctypes.addressof(pointers)
            a.cache_count = len(addresses)
        elif page is None or blocks is None:
            raise ValueError("without caches, page and blocks are needed")
        else:
            a.page, a.blocks = _page(page), int(blocks)
        if a.blocks < 1 or a.blocks * a.page > 2**31 - 1 or a.width * a.page > 2**31 - 1:
            raise ValueError("the cache and a table row must span 1 to 2^31 - 1 tokens")
        i32 = lambda *s: torch.empty(*s, dtype=torch.int32, device=dev)  # noqa: E731
        res = CommitResult(i32(R, MAX_NODES), i32(R, MAX_NODES), i32(R), i32(R), i32(R), i32(R), i32(R), i32(R))
        for field in ("path", "ids", "accepted", "count", "pending", "stop", "lengths", "status"):
            setattr(a, field, getattr(res, field).data_ptr())
        a.requests, a.tokens = R, n
        self._setup("dsr_commit_tree", a, dev, res,
                    (parents, tokens, sampled, offsets, kv_lengths, table, output_limit, eos_offsets, eos_ids,
                     pointers, *before, *caches, *vars(res).values()))


def commit_tree(parents, tokens, sampled, offsets, kv_lengths, table, caches, *, output_limit, eos_offsets=None,
                eos_ids=None, page: int | None = None, blocks: int | None = None, lengths=None, pending=None,
                plan_status=None) -> CommitResult:
    """The accepted path of each request's drafted tree, and its cache rows
    moved together in every one of ``caches`` (once in one that is listed twice,
    as keys that are also the values).

    ``tokens`` and ``sampled`` (int32) are each node's drafted token and the
    target's token drawn after it (``batch.sample_rows`` over the nodes' rows:
    the path then has exactly the target's distribution).  From node 0, the
    first child whose token was drawn is accepted, and so on; ids, stops and
    pending token follow ``verify_drafts``.  ``lengths`` of the result are the
    next step's ``lengths``.

    ``lengths`` (those given to ``plan_blocks``), ``pending`` (the pending
    tokens before the step) and ``plan_status`` (``plan_blocks``'s status), all
    int32 ``[requests]``, come together.  With them a request that the plan
    refused, or that has a status here, keeps its length and pending token for
    a later step, and one without new tokens its pending token.  Without them
    it gets length 0, or none pending: a loop whose pool can run short needs
    them."""
    return PreparedCommit(parents, tokens, sampled, offsets, kv_lengths, table, caches, output_limit=output_limit,
                          eos_offsets=eos_offsets, eos_ids=eos_ids, page=page, blocks=blocks, lengths=lengths,
                          pending=pending, plan_status=plan_status, upload=False).launch()
