"""dsr_fork_pages against the host oracle: tables, counts, pool and every byte
of the caches."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import branches
from oracle import branch_oracle as O
from tests.branch_util import Pages, caches_of, copied, far_apart
from tests.tree_util import i32

pytestmark = pytest.mark.gpu
FIELDS = ("table", "held", "lengths", "shared", "pool", "state", "status", "source_status")


def check(p, parents, caches=(), out=None, **kw):
    want = O.fork(p.lengths, parents, p.table, p.held, p.shared, p.pool, p.state, p.blocks, p.page)
    after = copied(caches, want["copies"])
    args = p.tensors("lengths") + [i32(parents)] + p.tensors("table", "held", "shared", "pool", "state")
    if not caches:
        kw = dict(page=p.page, blocks=p.blocks, **kw)
    res = branches.fork_pages(*args, caches, out=out, **kw)
    for f in FIELDS:
        np.testing.assert_array_equal(getattr(res, f).cpu().numpy(), want[f], err_msg=f)
    for x, y in zip(caches, after):
        assert torch.equal(x, y)
    return res, want, args


def consistent(p, want, live=None):
    """The counts are those of the tables; no page is both held and free."""
    holders = np.zeros(p.blocks, int)
    for row, n in zip(want["table"], want["held"]):
        holders[row[:n]] += 1
    np.testing.assert_array_equal(np.maximum(holders - 1, 0), want["shared"])
    head, count = want["state"]
    free = {int(want["pool"][(head + i) % len(want["pool"])]) for i in range(count)}
    assert len(free) == count and not free & set(np.flatnonzero(holders))
    assert count + (holders > 0).sum() == p.blocks - p.first


@pytest.mark.parametrize("rows,family,page,longest", [(1, 1, 16, 40), (8, 4, 16, 100), (32, 8, 1, 30), (40, 5, 64, 900),
                                                      (130, 2, 8, 64), (7, 7, 128, 127), (1100, 4, 4, 20)])
def test_a_step_of_beams(rows, family, page, longest):
    rng = np.random.default_rng([rows, family, page])
    p = Pages(rng, rng.integers(0, longest + 1, rows), family, page, spare=rows, extra=1)
    parents = np.arange(rows) // family * family + rng.integers(0, family, rows)
    parents = np.where(rng.random(rows) < 0.1, -1, np.minimum(parents, rows - 1))
    res, want, _ = check(p, parents, caches_of(rng, p, 3, 2, 16))
    consistent(p, want)


def test_steps_one_after_the_other():
    """Rows that go on, end and share for many steps: the counts stay those of the tables."""
    rng = np.random.default_rng(1)
    p = Pages(rng, [37, 50, 5, 0, 64, 63], 3, 8, spare=40)
    for step in range(12):
        rows = int(rng.integers(1, 14))
        parents = rng.integers(-1, len(p.lengths), rows)
        res, want, _ = check(p, parents, caches_of(rng, p, 1, 1, 8))
        consistent(p, want)
        p.table, p.held, p.lengths = want["table"], np.array(want["held"]), np.array(want["lengths"])
        p.shared, p.pool, p.state = want["shared"], want["pool"], np.array(want["state"])


@pytest.mark.parametrize("sources,rows", [(1, 64), (4, 3), (3, 50), (5, 0), (0, 5), (0, 0)])
def test_more_and_fewer_rows(sources, rows):
    rng = np.random.default_rng([sources, rows])
    p = Pages(rng, rng.integers(1, 60, sources), 1, 16, spare=70)
    parents = rng.integers(0, sources, rows) if sources else np.full(rows, -1)
    _, want, _ = check(p, parents, caches_of(rng, p, 2, 1, 8))
    consistent(p, want)


@pytest.mark.parametrize("by_head", [False, True])
@pytest.mark.parametrize("kv,dim,dtype", [(1, 8, "bf16"), (8, 128, "bf16"), (3, 96, "f16"), (2, 80, "f32")])
def test_caches_of_any_shape(kv, dim, dtype, by_head):
    rng = np.random.default_rng([kv, dim])
    p = Pages(rng, [45, 17, 31], 1, 32, spare=12)
    check(p, [0, 0, 0, 1, 2, 2, 1], caches_of(rng, p, 2, kv, dim, dtype, by_head))


@pytest.mark.parametrize("count", [0, 1, 128, 129, 300])
def test_many_caches(count):
    rng = np.random.default_rng(count)
    p = Pages(rng, [9, 30, 2], 1, 4, spare=12)
    parents = [0, 0, 2, 2, 1, 0]
    caches = caches_of(rng, p, count, 2, 16)
    again, kw = [t.clone() for t in caches], {} if count else dict(page=p.page, blocks=p.blocks)
    res, want, _ = check(p, parents, caches)
    args = p.tensors("lengths") + [i32(parents)] + p.tensors("table", "held", "shared", "pool", "state")
    other = branches.PreparedFork(*args, again + again, **kw).launch()  # one listed twice is moved once
    assert all(torch.equal(getattr(res, f), getattr(other, f)) for f in FIELDS)
    assert all(torch.equal(x, y) for x, y in zip(caches, again))


@pytest.mark.parametrize("free", [0, 1, 3])
def test_a_pool_that_runs_short(free):
    """Rows that lack a page are refused, ones that need none are not."""
    rng = np.random.default_rng(free)
    p = Pages(rng, [20, 16, 33], 1, 16, spare=free)
    _, want, _ = check(p, [0, 0, 1, 1, 2, 2, 0, 0, 1], caches_of(rng, p, 1, 1, 8))
    assert want["status"].count(O.E_BLOCKS) == max(0, 4 - free)


def test_a_pool_that_is_none():
    rng = np.random.default_rng(5)
    for state in ([-1, 3], [0, 1000], [1000, 0], [0, -1]):
        p = Pages(rng, [20, 16], 1, 16, spare=6)
        p.state = np.array(state, np.int32)
        check(p, [0, 0, 1, 1])


def test_rows_and_sources_out_of_bounds():
    rng = np.random.default_rng(6)
    p = Pages(rng, [20, 16, 33, 40, 8], 1, 16, spare=9)
    p.lengths[0] = -1
    p.held[1] = p.table.shape[1] + 1
    p.lengths[2] = 16 * p.held[2] + 1
    p.held[4] = -3
    check(p, [0, 1, 2, 3, 4, 3, -1, -2, 5, 1 << 30, -(1 << 31)], caches_of(rng, p, 1, 1, 8))


def test_pages_outside_the_cache():
    rng = np.random.default_rng(7)
    p = Pages(rng, [40, 40, 40], 1, 16, spare=9)
    p.table[0, 0], p.table[1, 2], p.table[2, 1] = -1, p.blocks, 1 << 30
    at = int(p.state[0])
    p.pool[at] = -5  # the first page that is handed out
    check(p, [0, 0, 1, 1, 2, 2], caches_of(rng, p, 1, 1, 8))
    check(p, [-1, -1, -1], caches_of(rng, p, 1, 1, 8))


def test_the_largest_batch():
    rng = np.random.default_rng(8)
    n = 16384
    p = Pages(rng, rng.integers(0, 20, n), 4, 8, spare=n)
    _, want, _ = check(p, rng.integers(-1, n, n))
    consistent(p, want)


def test_many_pages():
    """More pages than one workgroup counts the bits of."""
    rng = np.random.default_rng(9)
    p = Pages(rng, rng.integers(0, 3000, 64), 4, 1, spare=64, first=3)
    assert p.blocks > 2 * 32768
    _, want, _ = check(p, rng.integers(-1, 64, 64), caches_of(rng, p, 1, 1, 8))
    consistent(p, want)


def test_caches_past_32_bits():
    rng = np.random.default_rng(12)
    p = Pages(rng, [37, 50, 5, 63, 64, 30], 3, 8, spare=20)
    cache = far_apart(caches_of(rng, p, 1, 2, 16)[0])
    check(p, [0, 0, 1, 3, 3, 3, 5, 5, 2, 2], [cache])


def test_given_results_leave_the_inputs():
    rng = np.random.default_rng(10)
    p = Pages(rng, [20, 16, 33], 3, 16, spare=9)
    parents = [0, 0, 2, 2]
    out = dict(shared=torch.empty(p.blocks, dtype=torch.int32, device="cuda"), state=i32([7, 7]),
               table=torch.empty(4, 2 * p.table.shape[1], dtype=torch.int32, device="cuda")[:, :p.table.shape[1]])
    res, want, args = check(p, parents, caches_of(rng, p, 1, 1, 8), out=out)
    assert torch.equal(args[4], i32(p.shared)) and torch.equal(args[6], i32(p.state))
    assert res.table is out["table"]


def test_a_prepared_call_in_a_graph():
    rng = np.random.default_rng(11)
    p = Pages(rng, [20, 16, 33, 50], 2, 16, spare=12)
    caches = caches_of(rng, p, 140, 1, 16)
    start = [t.clone() for t in caches]
    t = {n: x for n, x in zip(("lengths", "table", "held", "shared", "pool", "state"),
                              p.tensors("lengths", "table", "held", "shared", "pool", "state"))}
    parents = i32([0, 1, 2, 3])
    call = branches.PreparedFork(t["lengths"], parents, t["table"], t["held"], t["shared"], t["pool"], t["state"],
                                 caches, upload=False)
    call.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call.launch()
    for turn in range(4):
        now = rng.integers(-1, 4, 4)
        parents.copy_(i32(now))
        for n in ("shared", "pool", "state"):
            t[n].copy_(i32(getattr(p, n)))
        for x, s in zip(caches, start):
            x.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        want = O.fork(p.lengths, now, p.table, p.held, p.shared, p.pool, p.state, p.blocks, p.page)
        for f in FIELDS:
            np.testing.assert_array_equal(getattr(got, f).cpu().numpy(), want[f], err_msg=f"{f} {turn}")
        assert all(torch.equal(x, y) for x, y in zip(caches, copied(start, want["copies"]))), turn


def test_refusals():
    rng = np.random.default_rng(12)
    p = Pages(rng, [20, 16, 33], 3, 16, spare=9)
    names = ("lengths", "table", "held", "shared", "pool", "state")
    good = dict(zip(names, p.tensors(*names)), parents=i32([0, 1, 2]), caches=caches_of(rng, p, 2, 2, 16))

    def call(out=None, **kw):
        a = {**good, **kw}
        return branches.fork_pages(a["lengths"], a["parents"], a["table"], a["held"], a["shared"], a["pool"],
                                   a["state"], a["caches"], out=out)

    c = good["caches"][0]
    for bad in (dict(lengths=good["lengths"].long()), dict(held=good["held"][:2]), dict(shared=good["shared"][1:]),
                dict(state=i32([0])), dict(table=good["table"][:2]), dict(caches=[]), dict(caches=[c[:, :12]]),
                dict(caches=[c, c[1:]]), dict(caches=[c, c.float()]), dict(caches=[c[..., :4]]),
                dict(out=dict(table=good["table"])), dict(out=dict(held=good["held"])),
                dict(out=dict(lengths=good["parents"])), dict(out=dict(state=i32([0, 1, 2]))),
                dict(out=dict(shared=good["pool"])), dict(out=dict(pool=good["pool"]))):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(TypeError):
        call(lengths=good["lengths"].cpu())
