"""Inputs shared by the tests of decoding with several branches a request."""
import numpy as np
import torch

from tests.tree_util import DTYPES, Step, i32


class Pages:
    """Rows in families of which each shares some of its first pages, and the
    pool of the other pages."""

    def __init__(self, rng, lengths, family, page, spare=3, first=0, width=None, extra=0):
        self.lengths = np.array(lengths, np.int32)
        self.page, self.first = page, first
        need = [-(-n // page) + int(rng.integers(0, extra + 1)) for n in lengths]
        self.blocks = first + sum(need) + spare
        width = width or max(need, default=0) + 2
        free = list(first + rng.permutation(self.blocks - first))
        self.table = np.full((len(lengths), width), -1, np.int32)
        self.shared = np.zeros(self.blocks, np.int32)
        self.held = np.array(need, np.int32)
        for at in range(0, len(lengths), family):
            rows = range(at, min(at + family, len(lengths)))
            common = int(rng.integers(0, min(lengths[r] // page for r in rows) + 1))
            both = [free.pop() for _ in range(common)]
            self.shared[both] = len(rows) - 1
            for r in rows:
                self.table[r, :need[r]] = both + [free.pop() for _ in range(need[r] - common)]
        size = self.blocks - first
        self.pool = np.full(size, -1, np.int32)
        head = int(rng.integers(0, size))
        self.pool[(head + np.arange(len(free))) % size] = free
        self.state = np.array([head, len(free)], np.int32)

    def tensors(self, *names):
        return [i32(getattr(self, n)) for n in names]


def caches_of(rng, p, count, kv, dim, dtype="bf16", by_head=False):
    shape = (p.blocks, kv, p.page, dim) if by_head else (p.blocks, p.page, kv, dim)
    made = [torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).cuda().to(DTYPES[dtype])
            for _ in range(count)]
    return [t.transpose(1, 2) for t in made] if by_head else made


def far_apart(cache):
    """The cache with its pages spread over more than 2^32 bytes."""
    blocks, *page = cache.shape
    elements = cache[0].numel()
    step = max(elements, ((5 << 30) // cache.element_size() // blocks + 127) // 128 * 128)
    strides = [elements // page[0], page[2], 1]
    far = torch.empty((blocks - 1) * step + elements, dtype=cache.dtype, device=cache.device)
    return far.as_strided(cache.shape, (step, *strides)).copy_(cache)


def copied(caches, copies):
    """The caches after the copies (from, to, tokens)."""
    out = []
    for old in caches:
        now = old.clone()
        for a, b, n in copies:
            now[b, :n] = old[a, :n]
        out.append(now)
    return out


class PrefixStep(Step):
    """Requests in groups that share the pages of a prefix; then `alone` ones."""

    def __init__(self, rng, family, prefix, new, own, heads, kv, dim, page, dtype, alone=0, **kw):
        groups = len(prefix)
        assert len(new) == len(own) == groups * family + alone
        common = [p for p in prefix for _ in range(family)] + [0] * alone
        super().__init__(rng, new, [c + o for c, o in zip(common, own)], heads, kv, dim, page, dtype, **kw)
        self.prefix = np.array(prefix, np.int32)
        self.groups = np.arange(groups + 1, dtype=np.int32) * family
        for g in range(groups):
            n = prefix[g] // page
            self.table[g * family:(g + 1) * family, :n] = self.table[g * family, :n]
            if prefix[g] % page:  # the same tokens on pages of their own
                first = self.table[g * family, n]
                for r in range(g * family + 1, (g + 1) * family):
                    for cache in (self.k, self.v):
                        cache[int(self.table[r, n]), :prefix[g] % page] = cache[int(first), :prefix[g] % page]

    def prefix_args(self):
        args, vis = self.args()
        return (*args, i32(self.groups, self.dev), i32(self.prefix, self.dev)), vis
