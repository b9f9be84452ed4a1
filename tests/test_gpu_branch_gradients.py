"""fork_pages and compact_pages write caches in place: ones that require a
gradient, which would be wrong afterwards without a word, are refused."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import branches
from tests.branch_util import Pages, caches_of
from tests.tree_util import i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", [0, 2])
def test_caches_that_require_a_gradient(which):
    rng = np.random.default_rng(1)
    p = Pages(rng, [20, 16, 33], 1, 16, spare=9)
    caches = caches_of(rng, p, 3, 2, 16)
    lengths, table, held, shared, pool, state = p.tensors("lengths", "table", "held", "shared", "pool", "state")

    def calls():
        yield lambda: branches.fork_pages(lengths, i32([0, 0, 2]), table, held, shared, pool, state, caches)
        yield lambda: branches.PreparedFork(lengths, i32([0, 0, 2]), table, held, shared, pool, state, caches)
        yield lambda: branches.compact_pages(table, held, pool, state, caches, shared=shared)
        yield lambda: branches.PreparedCompact(table, held, pool, state, caches, shared=shared)

    caches[which].requires_grad_()
    before = [t.detach().clone() for t in (*caches, table, held, shared, pool, state)]
    for call in calls():
        with pytest.raises(ValueError, match="gradients"):
            call()
    assert all(torch.equal(a, b) for a, b in zip(before, (*caches, table, held, shared, pool, state)))
    with torch.no_grad():
        for call in calls():
            call()
    leaf, caches[which] = caches[which], caches[which] * 1  # one that comes of a leaf
    for call in calls():
        with pytest.raises(ValueError, match="gradients"):
            call()
    caches[which] = leaf.detach()
    for call in calls():
        call()
