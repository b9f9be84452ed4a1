"""dsr_tree_attention within the bound of its own roundings
(tests/tree_exact.py), in every kernel: few rows, 32, 64 and 128 rows, whole
and in parts."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import tree
from tests import tree_exact
from tests.tree_util import Step

pytestmark = pytest.mark.gpu

CASES = [  # new tokens, contexts, heads, kv heads, dim, table columns to spare
    ([1], [3], 8, 2, 64, 0), ([4], [3], 8, 2, 128, 0), ([4, 1], [3, 700], 8, 2, 256, 0), ([5, 2], [2500, 9], 4, 1, 192, 0),
    ([1], [6000], 8, 1, 128, 0),
    ([3, 5], [600, 4], 8, 1, 64, 1 << 17), ([3, 5], [600, 4], 8, 1, 128, 1 << 17), ([3, 5], [4, 600], 8, 1, 96, 1 << 17),
    ([12, 9], [300, 4], 4, 1, 192, 1 << 17), ([12, 9], [4, 300], 4, 1, 256, 1 << 17),
    ([40, 21], [300, 4], 4, 1, 64, 1 << 17), ([40, 21], [300, 4], 4, 1, 128, 1 << 17),
    ([40, 33], [4, 300], 4, 1, 192, 1 << 17), ([40, 33], [4, 300], 4, 1, 256, 1 << 17),
    ([2] * 70, [20] * 70, 32, 8, 64, 0), ([2] * 70, [20] * 70, 32, 8, 128, 0), ([1] * 70, [20] * 70, 32, 8, 256, 0),
]


@pytest.mark.parametrize("new,ctx,heads,kv,dim,columns", CASES)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("trees,spread", [(True, 1.0), (False, 2.0)])
def test_within_its_roundings(new, ctx, heads, kv, dim, columns, dtype, trees, spread):
    rng = np.random.default_rng([sum(new), sum(ctx), dim, trees])
    step = Step(rng, new, ctx, heads, kv, dim, 16, dtype, trees, spread=spread)
    step.table = np.pad(step.table, ((0, 0), (0, columns)), constant_values=-1)
    args, vis = step.args()
    res = tree.tree_attention(*args, visible=vis, lse=True)
    tree_exact.check(step, res, dtype)
    assert not res.status.any()
