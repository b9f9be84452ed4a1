"""dsr_fork_pages with counts that are not those of the tables: which pages go
back to the pool follows from the counts afterwards, not from the order in which
sources change them."""
import numpy as np
import pytest

from oracle import branch_oracle as O
from tests.branch_util import Pages
from tests.test_gpu_branch_fork import check


def families(rng, kinds, others=0):
    """Sources of one full page each, in groups that hold the same one, of which
    `shared` knows a single holder; the children of each."""
    p = Pages(rng, [16] * (sum(map(len, kinds)) + others), 1, 16, spare=5)
    at = 0
    for children in kinds:
        p.table[at:at + len(children), 0] = p.table[at, 0]
        at += len(children)
    parents = [s for s, n in enumerate(c for children in kinds for c in children) for _ in range(n)]
    return p, parents + list(range(at, at + others))


KINDS = [[0, 3], [3, 0], [0, 0, 1], [0, 3, 0, 0], [3, 0, 0, 0], [0, 0, 0, 3], [2, 0, 0], [0, 2, 0], [1, 0], [0, 0]]


@pytest.mark.gpu
@pytest.mark.parametrize("times,others", [(1, 0), (40, 0), (40, 900)])
def test_the_order_of_sources_does_not_matter(times, others):
    rng = np.random.default_rng([times, others])
    kinds = [KINDS[i] for i in rng.permutation(len(KINDS) * times) % len(KINDS)]
    p, parents = families(rng, kinds, others)
    res, _, _ = check(p, parents)
    at = 0
    for children in kinds:  # one holder less than there are, whoever goes first
        page = p.table[at, 0]
        left = sum(n - 1 for n in children)
        assert int(res.shared[page]) == max(left, 0), children
        held = res.pool[(int(p.state[0]) + int(p.state[1]) + np.arange(len(res.pool))) % len(res.pool)]
        assert (page in held[:int(res.state[1]) - int(p.state[1])]) == (left < 0), children
        at += len(children)


def test_the_oracle_does_not_mind_the_order():
    for children in KINDS:
        freed = set()
        for order in (children, children[::-1], sorted(children)):
            p, parents = families(np.random.default_rng(1), [order])
            d = O.fork(p.lengths, parents, p.table, p.held, p.shared, p.pool, p.state, p.blocks, p.page)
            freed.add((d["state"][1] - p.state[1], int(d["shared"][p.table[0, 0]])))
        left = sum(n - 1 for n in children)
        assert freed == {(int(left < 0), max(left, 0))}, children
