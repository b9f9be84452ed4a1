"""Inputs and bounds shared by the tests of the tree-speculative operators."""
import numpy as np
import torch

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# Unit roundoff 2^-p of a type with p significant bits: the largest relative error of one rounding.
ROUND = {"bf16": 2.0**-8, "f16": 2.0**-11, "f32": 2.0**-24}


def random_tree(rng, n, back=6):
    return [-1] + [max(0, i - int(rng.integers(1, back + 1))) for i in range(1, n)] if n else []


def random_table(rng, pages, blocks, spare=0):
    """A block table with pages[r] different pages per row (-1 behind them)."""
    perm = rng.permutation(blocks)
    width = max(1, max(pages, default=1) + spare)
    table = np.full((len(pages), width), -1, np.int32)
    at = 0
    for r, p in enumerate(pages):
        table[r, :p] = perm[at:at + p]
        at += p
    return table, perm[at:]


def i32(x, dev="cuda"):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(x, np.int64).astype(np.int32))).to(dev)


class Step:
    """Random paged caches and new tokens for the attention tests."""

    def __init__(self, rng, new, ctx, heads, kv, dim, page, dtype, trees=False, by_head=False, dev="cuda", spread=1.0):
        self.page, self.kv, self.dim = page, kv, dim
        total = [c + n for c, n in zip(ctx, new)]
        pages = [-(-t // page) for t in total]
        blocks = max(1, sum(pages) + 2)
        self.table, _ = random_table(rng, pages, blocks, spare=1)
        self.offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.kv_lengths = np.array(total, np.int32)
        n = int(self.offsets[-1])
        shape = (blocks, kv, page, dim) if by_head else (blocks, page, kv, dim)
        t = DTYPES[dtype]

        def make(*s):
            return torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(dev).to(t)

        self.k, self.v, self.q = make(*shape), make(*shape), (make(n, heads, dim).float() * spread).to(t)
        if by_head:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.visible = None
        if trees:
            from oracle import tree_oracle as O
            words = []
            for m in new:
                par = random_tree(rng, m)
                words += [sum(1 << p for p in O.ancestors(par, i)) for i in range(m)]
            self.visible = np.array(words, np.uint64).view(np.int64)
        self.dev = dev

    def args(self):
        vis = None if self.visible is None else torch.from_numpy(self.visible.copy()).to(self.dev)
        return (self.q, self.k, self.v, i32(self.table, self.dev), i32(self.offsets, self.dev),
                i32(self.kv_lengths, self.dev)), vis

    def host(self):
        f = lambda x: x.cpu().float().numpy()  # noqa: E731
        return f(self.q), f(self.k), f(self.v), self.table, self.offsets, self.kv_lengths, self.visible


def attention_bound(dtype, out, size, q, k, scale, kv):
    """Largest error of the kernel's output against the exact one, per element.

    Each weight and the output are rounded to the type (u each; the weights'
    share scales with sum p |v|); a score carries at most dim float32 rounding
    errors of a sum below |q| |k| scale, a few ulps of the exponential, and the
    sums over the tokens one float32 rounding per addition of at most 64 in a
    row (32-token tiles, four waves, chunks; counted generously)."""
    u = ROUND[dtype]
    dim = q.shape[-1]
    top = np.abs(q).max() * np.sqrt(dim) * np.abs(k).max() * np.sqrt(dim) * abs(scale)
    f32 = 2.0**-24 * (dim * top + 8 * top + 64 + kv / 32)
    tiny = 2.0**-25 / 2.0**7 * kv * 8 if dtype == "f16" else 0.0  # weights below f16's normal numbers
    return (u + 2 * f32 + tiny) * size * 1.01 + u * np.abs(out) * 1.01 + 1e-7
