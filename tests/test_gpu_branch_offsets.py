"""dsr_prefix_attention with offsets that descend: every request is refused, no
row and no status is left as it was."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import branches
from tests.branch_util import PrefixStep
from tests.tree_exact import check
from tests.tree_util import i32

pytestmark = pytest.mark.gpu


def launch(args, vis=None):
    p = branches.PreparedPrefixAttention(*args, visible=vis, lse=True)
    p.result.out.fill_(9)
    p.result.lse.fill_(9)
    p.result.status.fill_(77)
    return p.launch()


@pytest.mark.parametrize("offsets", [[0, 5, 2, 8], [3, 1, 8, 8], [0, 8, 0, 8], [8, 5, 3, 0], [0, 3, 8, 7], [-5, 3, -5, 8]])
@pytest.mark.parametrize("groups", [[0, 3], [0, 2, 3], [1, 3], [3, 3]])
@pytest.mark.parametrize("heads,dim", [(2, 64), (32, 128), (16, 256)])
def test_every_request_is_refused(offsets, groups, heads, dim):
    rng = np.random.default_rng(1)
    step = PrefixStep(rng, 3, [64], [3, 3, 2], [20] * 3, heads, 2, dim, 16, "bf16")
    step.groups, step.prefix = np.array(groups, np.int32), np.full(len(groups) - 1, 64, np.int32)
    args, _ = step.prefix_args()
    res = launch((*args[:4], i32(offsets), *args[5:]))
    assert res.status.tolist() == [16] * 3
    assert not res.out.any() and torch.isneginf(res.lse).all()
    res = launch(args)  # the same call with its own offsets
    assert not res.status.any()
    check(step, res, "bf16")


def test_many_requests():
    """More than every workgroup looks over for itself; one pair of offsets changed places."""
    rng = np.random.default_rng(2)
    R = 1500
    step = PrefixStep(rng, 500, [8] * 3, [1] * R, [3] * R, 2, 1, 64, 8, "bf16")
    args, _ = step.prefix_args()
    offsets = step.offsets.copy()
    offsets[[1400, 1401]] = offsets[[1401, 1400]]
    res = launch((*args[:4], i32(offsets), *args[5:]))
    assert (res.status == 16).all() and not res.out.any() and torch.isneginf(res.lse).all()


def test_offsets_past_the_tokens_may_descend():
    """Held to the tokens that there are they do not."""
    rng = np.random.default_rng(3)
    step = PrefixStep(rng, 3, [64], [3, 5, 0], [20] * 3, 4, 2, 64, 16, "bf16")
    args, _ = step.prefix_args()
    res = launch((*args[:4], i32([-2, 3, 100, 90]), *args[5:]))
    assert not res.status.any()
    check(step, res, "bf16")
