"""dsr_compact_pages against the host oracle."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import branches
from oracle import branch_oracle as O
from tests.branch_util import Pages, caches_of, copied, far_apart
from tests.tree_util import i32

pytestmark = pytest.mark.gpu
FIELDS = ("table", "shared", "pool", "state", "remap", "status")


def check(p, caches=(), shared=True, out=None, in_place=True):
    want = O.compact(p.table, p.held, p.shared if shared else None, p.pool, p.state, p.blocks, p.page, p.first)
    after = copied(caches, want["copies"])
    table, held, pool, state = p.tensors("table", "held", "pool", "state")
    kw = {} if caches else dict(page=p.page, blocks=p.blocks)
    res = branches.compact_pages(table, held, pool, state, caches, shared=i32(p.shared) if shared else None,
                                 first=p.first, out=out, **kw)
    for f in FIELDS:
        if f != "shared" or shared:
            np.testing.assert_array_equal(getattr(res, f).cpu().numpy(), want[f], err_msg=f)
    assert all(torch.equal(x, y) for x, y in zip(caches, after))
    if out is None:
        assert res.table is table and res.pool is pool and res.state is state
    return res, want


@pytest.mark.parametrize("rows,page,longest,spare,first", [(1, 16, 30, 0, 0), (5, 16, 100, 1, 0), (16, 8, 200, 300, 1),
                                                           (40, 64, 900, 90, 7), (3, 1, 12000, 9000, 40),
                                                           (1, 1, 3, 100000, 0), (700, 4, 9, 2000, 33)])
@pytest.mark.parametrize("shared", [False, True])
def test_matches_the_oracle(rows, page, longest, spare, first, shared):
    rng = np.random.default_rng([rows, page, spare, first])
    p = Pages(rng, rng.integers(0, longest + 1, rows), 4, page, spare=spare, first=first, extra=1)
    _, want = check(p, caches_of(rng, p, 3, 1, 8), shared)
    # What each row reads afterwards is what it read before.
    assert sorted(want["pool"][:want["state"][1]]) == want["pool"][:want["state"][1]]
    again = Pages.__new__(Pages)
    again.__dict__ = dict(p.__dict__, table=want["table"], pool=want["pool"], state=want["state"],
                          shared=want["shared"] if shared else p.shared)
    _, twice = check(again, (), shared)
    assert not twice["copies"]


def test_nothing_held_and_everything_held():
    rng = np.random.default_rng(1)
    p = Pages(rng, [0, 0, 0], 1, 16, spare=50)
    check(p, caches_of(rng, p, 1, 1, 8))
    p = Pages(rng, [64, 64, 64], 1, 16, spare=0 + 1)
    check(p, caches_of(rng, p, 1, 1, 8))
    none = Pages(rng, [], 1, 16, spare=20, width=3)
    check(none, caches_of(rng, none, 1, 1, 8))


def test_pages_before_the_first_stay():
    """Rows may hold pages that no pool gave out: they are left alone."""
    rng = np.random.default_rng(2)
    p = Pages(rng, [64, 40, 20], 1, 16, spare=30, first=6)
    p.table[0, 0], p.table[2, 1] = 2, 5
    check(p, caches_of(rng, p, 2, 1, 8))


def test_caches_past_32_bits():
    rng = np.random.default_rng(13)
    p = Pages(rng, [64, 40, 20, 90], 2, 8, spare=30, first=2)
    _, want = check(p, [far_apart(caches_of(rng, p, 1, 2, 16)[0])])
    assert want["copies"]


@pytest.mark.parametrize("count", [1, 128, 129, 300])
@pytest.mark.parametrize("by_head", [False, True])
def test_many_caches(count, by_head):
    rng = np.random.default_rng(count)
    p = Pages(rng, [9, 30, 2, 17], 1, 4, spare=30)
    caches = caches_of(rng, p, count, 2, 16, by_head=by_head)
    again = [t.clone() for t in caches]
    res, _ = check(p, caches)
    table, held, pool, state = p.tensors("table", "held", "pool", "state")
    other = branches.PreparedCompact(table, held, pool, state, again + again, shared=i32(p.shared)).launch()
    assert all(torch.equal(getattr(res, f), getattr(other, f)) for f in FIELDS)
    assert all(torch.equal(x, y) for x, y in zip(caches, again))


@pytest.mark.parametrize("row,held,page_id", [(0, -1, None), (2, 99, None), (1, None, -1), (1, None, 1 << 30),
                                              (2, None, "blocks")])
def test_rows_out_of_bounds_refuse_the_call(row, held, page_id):
    rng = np.random.default_rng(3)
    p = Pages(rng, [40, 40, 40], 1, 16, spare=30)
    if held is not None:
        p.held[row] = held
    else:
        p.table[row, 1] = p.blocks if page_id == "blocks" else page_id
    _, want = check(p, caches_of(rng, p, 1, 1, 8))
    assert any(want["status"])
    out = {f: torch.zeros_like(t) for f, t in zip(("table", "pool", "state", "shared"),
                                                  p.tensors("table", "pool", "state", "shared"))}
    check(p, caches_of(rng, p, 1, 1, 8), out=out)


def test_given_results_leave_the_inputs_and_a_graph():
    rng = np.random.default_rng(4)
    p = Pages(rng, rng.integers(0, 200, 9), 3, 16, spare=60, first=2)
    caches = caches_of(rng, p, 3, 2, 16)
    table, held, pool, state, shared = p.tensors("table", "held", "pool", "state", "shared")
    out = dict(table=torch.empty(9, 40, dtype=torch.int32, device="cuda")[:, 1:1 + table.shape[1]],
               pool=torch.empty_like(pool), state=torch.empty_like(state), shared=torch.empty_like(shared))
    want = O.compact(p.table, p.held, p.shared, p.pool, p.state, p.blocks, p.page, p.first)
    after = copied(caches, want["copies"])
    call = branches.PreparedCompact(table, held, pool, state, caches, shared=shared, first=2, out=out)
    call.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call.launch()
    for turn in range(3):  # the moved pages are as they were: the same again
        for t in (*out.values(), got.remap, got.status):
            t.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        for f in FIELDS:
            np.testing.assert_array_equal(getattr(got, f).cpu().numpy(), want[f], err_msg=f"{f} {turn}")
        assert all(torch.equal(x, y) for x, y in zip(caches, after)), turn
    for t, n in ((table, "table"), (pool, "pool"), (state, "state"), (shared, "shared")):
        assert torch.equal(t, i32(getattr(p, n))), n


def test_refusals():
    rng = np.random.default_rng(5)
    p = Pages(rng, [20, 16, 33], 3, 16, spare=9, first=1)
    table, held, pool, state, shared = p.tensors("table", "held", "pool", "state", "shared")
    c = caches_of(rng, p, 1, 2, 16)[0]

    def call(table=table, held=held, pool=pool, state=state, caches=(c,), first=1, **kw):
        return branches.compact_pages(table, held, pool, state, caches, first=first, **kw)

    for bad in (dict(table=table.long()), dict(held=held[:2]), dict(pool=pool[1:]), dict(first=0), dict(first=-1),
                dict(first=p.blocks), dict(state=i32([0])), dict(shared=shared[1:]), dict(caches=()),
                dict(caches=(c, c[..., :8])), dict(page=8), dict(blocks=p.blocks - 1),
                dict(out=dict(pool=shared)), dict(out=dict(shared=shared)), dict(out=dict(table=table[:, 1:])),
                dict(shared=shared, out=dict(remap=shared)), dict(out=dict(status=held))):
        with pytest.raises(ValueError):
            call(**bad)
