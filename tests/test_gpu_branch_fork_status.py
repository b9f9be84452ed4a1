"""dsr_fork_pages: a row whose tokens could not be copied has a status, though
every page of its own is one of the cache."""
import numpy as np
import pytest

from oracle import branch_oracle as O
from tests.branch_util import Pages, caches_of
from tests.test_gpu_branch_fork import check


@pytest.mark.gpu
@pytest.mark.parametrize("page_id", [-1, "blocks", 1 << 30])
@pytest.mark.parametrize("others", [0, 1200])
def test_a_page_that_cannot_be_copied(page_id, others):
    rng = np.random.default_rng(others)
    p = Pages(rng, [40, 40, 40] + [16] * others, 1, 16, spare=9)
    p.table[1, 2] = p.blocks if page_id == "blocks" else page_id  # source 1's unfilled page
    parents = [0, 0, 1, 1, 1, 2, 2] + list(range(3, 3 + others))
    res, want, _ = check(p, parents, caches_of(rng, p, 2, 1, 8))
    assert res.status.tolist()[:7] == [0, 0] + [O.E_BLOCK] * 3 + [0, 0]
    assert not res.status[7:].any() and res.source_status.tolist()[:3] == [0, O.E_BLOCK, 0]
    held = res.table[3:5, 2].tolist()  # pages of their own, of unknown tokens
    assert all(0 <= x < p.blocks for x in held) and res.lengths.tolist()[3:5] == [40, 40]


def test_the_oracle_says_so():
    fork = O.fork([5], [0, 0], [[0, 9]], [2], np.zeros(4, int), [1, 2, 3, -1], [0, 3], 4, 4)
    assert fork["status"] == [O.E_BLOCK, O.E_BLOCK] and fork["source_status"] == [O.E_BLOCK] and not fork["copies"]
