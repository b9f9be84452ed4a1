"""Token arrays longer than the step's tokens: rows of tree_attention that
belong to no request."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import tree
from tests.tree_util import Step, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,ctx,heads,kv,dim,columns", [
    ([1], [40], 4, 2, 64, 0),             # few rows, whole
    ([1, 1], [9000, 3], 8, 1, 128, 0),    # few rows, in parts
    ([3] * 70, [20] * 70, 64, 8, 128, 0),  # tiles of 128 rows
    ([3] * 5, [90] * 5, 8, 1, 128, 1 << 17),   # tiles of 32, roomy tables
    ([12] * 5, [90] * 5, 8, 2, 256, 1 << 17),  # tiles of 64
    ([0, 0], [0, 5], 4, 2, 64, 0),        # nobody has tokens
])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lead,behind", [(0, 1), (0, 200), (7, 3)])
def test_rows_of_no_request(new, ctx, heads, kv, dim, columns, dtype, lead, behind):
    rng = np.random.default_rng([sum(new), dim, lead, behind])
    step = Step(rng, new, ctx, heads, kv, dim, 16, dtype, trees=True)
    (q, k, v, table, offsets, kv_lengths), vis = step.args()
    table = torch.nn.functional.pad(table, (0, columns), value=-1)
    n = sum(new)
    want = tree.tree_attention(q, k, v, table, offsets, kv_lengths, visible=vis, lse=True)
    wide = torch.full((lead + n + behind, heads, dim), float("nan"), device="cuda", dtype=q.dtype)
    wide[lead:lead + n] = q
    seen = torch.full((lead + n + behind,), -1, device="cuda", dtype=torch.int64)
    seen[lead:lead + n] = vis
    call = tree.PreparedTreeAttention(wide, k, v, table, offsets + lead, kv_lengths, visible=seen, lse=True)
    for _ in range(2):
        call.result.out.fill_(float("nan"))
        call.result.lse.fill_(float("nan"))
        res = call.launch()
        inside = slice(lead, lead + n)
        outside = torch.tensor([i for i in range(lead + n + behind) if not lead <= i < lead + n], device="cuda")
        assert (res.out[outside] == 0).all() and torch.isneginf(res.lse[outside]).all()
        assert torch.allclose(res.out[inside].float(), want.out.float(), rtol=2**-7, atol=2**-9)
        assert torch.allclose(res.lse[inside], want.lse, rtol=1e-5, atol=1e-5)
        assert torch.equal(res.status, want.status)


def test_a_plan_with_spare_capacity():
    """The loop's own order: plan, attention, with more places than tokens."""
    rng = np.random.default_rng(1)
    pool, state = tree.page_pool(20)
    plan = tree.plan_blocks(i32([0, 0]), i32([3, 5]), i32(np.full((2, 4), -1)), i32([0, 0]), pool, state, blocks=20,
                            page=4, capacity=40, parents=i32([-1, 0, 1, -1, 0, 1, 2, 3] + [-1] * 32))
    cache = torch.from_numpy(rng.standard_normal((20, 4, 2, 64))).cuda().half()
    q = torch.from_numpy(rng.standard_normal((40, 4, 64))).cuda().half()
    out = torch.full_like(q, float("nan"))
    res = tree.tree_attention(q, cache, cache, plan.table, plan.offsets, plan.kv_lengths, visible=plan.visible, out=out)
    assert torch.isfinite(out).all() and not out[8:].any() and out[:8].any(-1).all() and not res.status.any()
