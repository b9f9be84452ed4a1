"""dsr_prefix_attention of groups whose first rows are empty, hundreds of them:
the row that leads is found, and finding it takes no time to speak of."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import branches, tree
from tests.branch_util import PrefixStep
from tests.tree_exact import check
from tests.tree_util import i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("family,groups,alone", [(700, 1, 0), (250, 2, 40), (1500, 1, 3), (400, 5, 0), (1, 1300, 0)])
@pytest.mark.parametrize("n,heads,dim", [(1, 4, 64), (9, 16, 128)])
def test_empty_rows_lead(family, groups, alone, n, heads, dim):
    rng = np.random.default_rng([family, groups, n])
    R = family * groups + alone
    new, own = np.zeros(R, int), np.zeros(R, int)
    for g in range(groups):  # the last rows of a group, or none
        live = g * family + family - 1 - np.arange(min(family, 3 if g != 1 else 0))
        new[live], own[live] = n, rng.integers(0, 50, len(live))
    new[R - alone:], own[R - alone:] = n, 7
    if groups == 1300:
        new[rng.random(R) < 0.9] = 0
    prefix = np.where(np.arange(groups) % 7 == 3, 0, 96 + 8 * (np.arange(groups) % 5))
    step = PrefixStep(rng, family, list(prefix), list(new), list(own), heads, 2, dim, 8, "bf16", alone)
    for r in np.flatnonzero(new == 0):
        step.table[r], step.kv_lengths[r] = -1, 0
    refused = int(np.flatnonzero(new > 0)[0])  # would lead, but its context is shorter than the prefix
    args, _ = step.prefix_args()
    res = branches.prefix_attention(*args, lse=True)
    assert not res.status.any()
    check(step, res, "bf16")
    want = tree.tree_attention(*args[:6], lse=True)
    step.kv_lengths[refused] = n + 1
    again = branches.prefix_attention(*step.prefix_args()[0], lse=True)
    status = np.zeros(R, int)
    status[refused] = 16 if refused < family * groups and prefix[refused // family] else 0
    assert again.status.tolist() == status.tolist()
    lo, hi = step.offsets[refused:refused + 2]
    rest = torch.ones(step.offsets[-1], dtype=torch.bool, device="cuda")
    rest[lo:hi] = False
    # Two results, each off by 2^-8 of itself and of the values' mean size (below 4 together).
    assert (again.out[rest].float() - want.out[rest].float()).abs().max() <= 2.0**-5
    assert (again.lse[rest] - want.lse[rest]).abs().max() <= 1e-5
    if status[refused]:
        assert not again.out[lo:hi].any() and torch.isneginf(again.lse[lo:hi]).all()


def fastest(new, prefix=256, own=8, page=16):
    """One group over a prefix, a token of the rows where `new` says so: the least of some times."""
    R, count, dev = new.numel(), int(new.sum()), "cuda"
    width = (prefix + own + 1 + page - 1) // page
    table = torch.arange(R * width, device=dev, dtype=torch.int32).view(R, width) % 4096
    table[:, :prefix // page] = torch.arange(prefix // page, device=dev)
    k, v = torch.randn(2, 4096, page, 2, 128, device=dev).to(torch.bfloat16)
    q = torch.randn(count, 8, 128, device=dev).to(torch.bfloat16)
    offsets = torch.cat([new.new_zeros(1), new.cumsum(0).int()]).to(dev)
    kv = ((prefix + own + 1) * new).int().to(dev)
    call = branches.PreparedPrefixAttention(q, k, v, table, offsets, kv, i32([0, R]), i32([prefix]))
    assert not call.launch().status.any()
    times = []
    for _ in range(7):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(4):
            call.launch()
        end.record()
        end.synchronize()
        times.append(begin.elapsed_time(end))
    return min(times)


@pytest.mark.parametrize("R", [1024, 2048, 16384])
def test_where_the_live_rows_are_does_not_matter(R):
    """Gone through one by one, the empty rows took 9 times a call's time of 1,024
    and 24 times that of 16,384 (now 1.1 and 1.6: the shares are looked for twice)."""
    at = torch.arange(R)
    first, last = fastest((at < 8).int()), fastest((at >= R - 8).int())
    assert last <= 4 * first, (first, last)
