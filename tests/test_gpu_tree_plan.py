"""dsr_plan_blocks against the host oracle: every output is a whole number and
must be equal."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import tree
from oracle import tree_oracle as O
from tests.tree_util import i32, random_table, random_tree

pytestmark = pytest.mark.gpu


def case(rng, R, new_hi, context, page, trees, ended=0.1, capacity_slack=0, short=False, spare_held=True):
    lengths = rng.integers(0, context + 1, R)
    added = rng.integers(0, new_hi + 1, R)
    added[rng.random(R) < ended] = -1
    held = -(-lengths // page)
    if spare_held:
        held = held + rng.integers(0, 3, R)  # pages kept from rejected tokens
    width = -(-(context + new_hi) // page) + 3
    blocks = int(held.sum()) + R * (-(-new_hi // page) + 1) + 3
    table, rest = random_table(rng, list(held), blocks)
    table = np.concatenate([table, np.full((R, max(0, width - table.shape[1])), -1, np.int32)], 1)
    size = blocks + 5
    pool = np.full(size, -1, np.int32)
    head = int(rng.integers(0, size))
    count = len(rest) if not short else min(len(rest), max(1, R // 2))
    pool[(head + np.arange(count)) % size] = rest[:count]
    capacity = max(1, int(added.clip(0).sum()) + capacity_slack)
    parents = None
    if trees:
        parents = np.concatenate([np.array(random_tree(rng, max(0, int(a))), np.int64) for a in added]
                                 + [np.full(max(0, capacity - int(added.clip(0).sum())), -1, np.int64)])[:capacity]
    return dict(lengths=lengths, added=added, table=table, held=held, pool=pool, state=[head, count], blocks=blocks,
                page=page, capacity=capacity, parents=parents)


def check(c, in_place=True):
    want = O.plan(**c)
    args = [i32(c[k]) for k in ("lengths", "added", "table", "held", "pool", "state")]
    before = [a.clone() for a in args]
    out = {} if in_place else dict(held=torch.empty_like(args[3]), state=torch.empty_like(args[5]))
    parents = None if c["parents"] is None else i32(c["parents"])
    call = tree.PreparedPlan(*args, blocks=c["blocks"], page=c["page"], capacity=c["capacity"], parents=parents,
                             out=out)
    for turn in range(1 if in_place else 2):  # out of place a call can be repeated
        res = call.launch()
        for key, w in want.items():
            if w is None:
                assert getattr(res, key) is None
                continue
            np.testing.assert_array_equal(getattr(res, key).cpu().numpy(), w, err_msg=key)
    for i in (0, 1) + (() if in_place else (3, 5)):
        assert torch.equal(args[i], before[i])
    return want


@pytest.mark.parametrize("R,new_hi,context,page", [(1, 1, 0, 16), (1, 1, 31, 16), (3, 7, 40, 8), (64, 1, 500, 16),
                                                   (65, 40, 300, 1), (256, 16, 200, 32), (300, 33, 90, 16),
                                                   (1500, 3, 60, 4), (7, 3000, 100, 128), (1, 9000, 17, 64)])
@pytest.mark.parametrize("trees", [False, True])
def test_plan_matches_oracle(R, new_hi, context, page, trees):
    if trees and new_hi > 64:
        pytest.skip("a tree has at most 64 nodes")
    rng = np.random.default_rng([R, new_hi, context, page, trees])
    want = check(case(rng, R, new_hi, context, page, trees))
    assert (want["status"] == 0).all()
    check(case(rng, R, new_hi, context, page, trees, capacity_slack=100, spare_held=False), in_place=False)


def test_many_empty_requests_between_tokens():
    rng = np.random.default_rng(5)
    c = case(rng, 9000, 0, 20, 16, False, ended=0.0)
    c["added"][[0, 3000, 8999]] = (2, 1, 70)
    c["capacity"] = 8192
    check(c)


@pytest.mark.parametrize("trees", [False, True])
@pytest.mark.parametrize("R", [40, 700])
def test_refusals(R, trees):
    """Pools that run out, token arrays too short, lengths out of bounds, page
    ids outside the cache: the others are served as if alone."""
    rng = np.random.default_rng([R, trees])
    c = case(rng, R, 30, 100, 8, trees, short=True, spare_held=False)
    want = check(c)
    assert (want["status"] == O.E_BLOCKS).any() and (want["status"] == 0).any()
    c = case(rng, R, 30, 100, 8, trees)
    c["capacity"] = max(1, c["capacity"] // 2)
    if trees:
        c["parents"] = c["parents"][:c["capacity"]]
    want = check(c)
    assert (want["status"] == O.E_CAPACITY).any()
    c = case(rng, R, 30, 100, 8, False)
    c["lengths"][0], c["added"][1], c["held"][2], c["held"][3] = -1, -2, -1, 10**6
    c["lengths"][4], c["added"][5] = 2**31 - 1, 2**31 - 1
    want = check(c)
    assert (want["status"][:6] == O.E_LENGTH).all()
    c = case(rng, R, 30, 100, 8, trees)
    c["pool"][:] = np.where(rng.random(len(c["pool"])) < 0.1, c["blocks"], c["pool"])
    want = check(c)
    assert (want["status"] == O.E_BLOCK).any()
    c = case(rng, R, 30, 100, 8, trees)
    c["state"] = [-3, 4]  # not a pool
    check(c)


def test_malformed_trees():
    rng = np.random.default_rng(9)
    c = case(rng, 30, 20, 50, 8, True, ended=0.0)
    c["added"][:] = np.maximum(c["added"], 2)
    c["capacity"] = int(c["added"].sum())
    c["parents"] = np.concatenate([random_tree(rng, int(a)) for a in c["added"]])
    off = np.concatenate([[0], np.cumsum(c["added"])])
    c["parents"][off[3] + 1] = 1      # its own parent
    c["parents"][off[7] + 1] = 5      # a later one
    c["parents"][off[9]] = -2
    c["parents"][off[11]:off[12]] = -1  # a forest is fine
    want = check(c)
    assert list(np.flatnonzero(want["status"])) == [3, 7, 9]
    c = case(rng, 3, 10, 50, 8, True, ended=0.0)
    c["added"][:] = (64, 65, 64)      # chains: the longest paths, and one node too many
    c["table"] = np.concatenate([c["table"], np.full((3, 20), -1, np.int32)], 1)
    c["pool"] = np.arange(100, dtype=np.int32)
    c["state"], c["blocks"], c["capacity"] = [90, 90], 100, 193
    c["parents"] = np.concatenate([np.arange(-1, n - 1) for n in (64, 65, 64)])
    want = check(c)
    assert list(want["status"]) == [0, O.E_TREE, 0]


def test_a_pool_through_many_steps():
    """Plans in place, lengths accepted or taken back between them, requests
    ending and starting again: pages are never shared or lost."""
    rng = np.random.default_rng(11)
    R, page, blocks = 20, 4, 300
    pool, state = tree.page_pool(blocks)
    held, lengths, table = i32(np.zeros(R)), np.zeros(R, int), i32(np.full((R, 40), -1))
    for step in range(40):
        added = rng.integers(0, 12, R)
        added[(rng.random(R) < 0.15) | (lengths + added > 150)] = -1
        res = tree.plan_blocks(i32(lengths), i32(added), table, held, pool, state, blocks=blocks, page=page,
                               capacity=max(1, int(added.clip(0).sum())))
        st, h, tab = res.status.cpu().numpy(), held.cpu().numpy(), table.cpu().numpy()
        assert (st == 0).all()
        head, count = state.tolist()
        free = pool.cpu().numpy()[(head + np.arange(count)) % blocks]
        owned = np.concatenate([tab[r, :h[r]] for r in range(R)] + [free])
        assert sorted(owned) == list(range(blocks))
        keep = np.where(added > 0, rng.integers(0, added.clip(0) + 1), 0)
        lengths = np.where(added < 0, 0, lengths + keep)


def test_no_requests_and_refused_arguments():
    z = i32([])
    res = tree.plan_blocks(z, z, torch.empty(0, 4, dtype=torch.int32, device="cuda"), z, i32([3, 4]), i32([0, 2]),
                           blocks=5, page=8, capacity=300)
    assert res.offsets.tolist() == [0] and res.state.tolist() == [0, 2]
    assert (res.slots == -1).all() and (res.owners == -1).all() and (res.positions == 0).all()
    one, tab = i32([1]), i32([[-1, -1]])
    good = dict(lengths=one, added=one, table=tab, held=i32([0]), pool=i32([0]), state=i32([0, 1]))
    kw = dict(blocks=1, page=8, capacity=4)
    tree.plan_blocks(*good.values(), **kw)
    for key, bad in (("lengths", one.long()), ("added", i32([1, 2])), ("table", tab.float()), ("held", one.cpu()),
                     ("pool", z), ("state", i32([0, 1, 2]))):
        with pytest.raises((TypeError, ValueError)):
            tree.plan_blocks(*dict(good, **{key: bad}).values(), **kw)
    for bad in (dict(kw, page=12), dict(kw, page=0), dict(kw, page=2048), dict(kw, blocks=0), dict(kw, capacity=0),
                dict(kw, blocks=2**30), dict(kw, parents=one), dict(kw, out=dict(nothing=one)),
                dict(kw, out=dict(slots=one))):
        with pytest.raises((TypeError, ValueError)):
            tree.plan_blocks(*good.values(), **bad)
