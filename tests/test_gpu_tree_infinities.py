"""Infinities and NaN in values: rows that see one hold what the sum would, in
the dimensions where it lies and with its sign; all others are as without it.
Keys stay finite, so that every row's weights do."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import tree
from tests import tree_exact
from tests.tree_util import Step

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")

CASES = [  # new tokens, contexts, heads, kv heads, dim, table columns to spare
    ([6], [70], 4, 2, 64, 0),               # few rows, whole
    ([6], [5000], 4, 2, 64, 0),             # few rows, in parts
    ([3], [4000], 4, 1, 128, 0), ([2], [300], 4, 2, 256, 0), ([7], [3000], 2, 1, 192, 0),
    ([5], [90], 4, 1, 64, 1 << 17),         # tiles of 32
    ([5], [5000], 4, 1, 128, 1 << 17),      # ... in parts
    ([12], [90], 4, 2, 256, 1 << 17), ([12], [2500], 4, 2, 192, 1 << 17),   # tiles of 64
    ([40], [70], 4, 2, 64, 1 << 17), ([40], [3000], 4, 1, 128, 1 << 17),    # tiles of 128
    ([50], [2000], 4, 1, 256, 1 << 17), ([50], [100], 4, 1, 192, 1 << 17),
    ([3] * 70, [20] * 70, 32, 8, 128, 0),   # tiles of 128, whole
]


def spoil(step, r, place, first=0, what=(INF, -INF, NAN)):
    """Dimensions first, first + 5, ... of a cached token's value become what[0], the next ones what[1], ..."""
    b, o = int(step.table[r, place // step.page]), place % step.page
    for i, x in enumerate(what):
        step.v[b, o, :, first + i::5] = x


def run(step, dtype):
    args, vis = step.args()
    return tree.tree_attention(*args, visible=vis, lse=True)


def made(new, ctx, heads, kv, dim, columns, dtype, trees, page=16):
    rng = np.random.default_rng([sum(new), sum(ctx), dim, trees])
    step = Step(rng, new, ctx, heads, kv, dim, page, dtype, trees)
    step.table = np.pad(step.table, ((0, 0), (0, columns)), constant_values=-1)
    return step


@pytest.mark.parametrize("new,ctx,heads,kv,dim,columns", CASES)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("trees", [True, False])
def test_new_tokens(new, ctx, heads, kv, dim, columns, dtype, trees):
    """A node in the middle, and the last one with other dimensions."""
    step = made(new, ctx, heads, kv, dim, columns, dtype, trees)
    spoil(step, 0, ctx[0] + new[0] // 2)
    spoil(step, 0, ctx[0] + new[0] - 1, first=1, what=(NAN, -INF, INF))
    if len(new) > 1:
        spoil(step, 33, ctx[33] + 1, what=(-INF, INF))
    out = tree_exact.check(step, run(step, dtype), dtype)
    assert np.isposinf(out).any() and np.isneginf(out).any() and np.isnan(out).any() and np.isfinite(out).any()


@pytest.mark.parametrize("new,ctx,heads,kv,dim,columns", CASES)
@pytest.mark.parametrize("back", [1, 20, 33, 64])
def test_context_tokens_near_its_end(new, ctx, heads, kv, dim, columns, back):
    """Every row sees them, some in steps that are looked through for the rows' own tokens."""
    step = made(new, ctx, heads, kv, dim, columns, "bf16", True)
    for r in range(0, len(new), 9):
        spoil(step, r, max(0, ctx[r] - back), what=(INF, -INF))
    out = tree_exact.check(step, run(step, "bf16"), "bf16")
    assert np.isinf(out).any() and np.isfinite(out).any()


@pytest.mark.parametrize("new,ctx,heads,kv,dim,columns", CASES)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("page", [1, 16])
def test_beside_a_page_outside_the_cache(new, ctx, heads, kv, dim, columns, dtype, page):
    """Its tokens are left out; what others hold still shows, wherever it lies.
    The first page, which is read in the place of one outside, is bad too."""
    step = made(new, ctx, heads, kv, dim, columns // (16 // page), dtype, True, page)
    spoil(step, 0, 2)
    spoil(step, 0, ctx[0] + new[0] // 2, first=1, what=(NAN, -INF, INF))
    used = np.isin(np.arange(step.k.shape[0]), step.table)
    first = step.table == 0
    if first.any():  # page 0 belongs to no request
        step.table[first] = int(np.flatnonzero(~used)[0])
        b = step.table[first][0]
        step.k[b], step.v[b] = step.k[0].clone(), step.v[0].clone()
    step.k[0], step.v[0] = NAN, INF
    step.table[0, (ctx[0] // 2) // page] = step.k.shape[0] + 5
    res = run(step, dtype)
    tree_exact.check(step, res, dtype)
    assert res.status[0] == tree.E_BLOCK and not res.status[1:].any()
