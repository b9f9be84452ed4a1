"""commit_tree as a call within a step: it does not wait for the stream, and it
can be captured."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import tree
from oracle import tree_oracle as O
from tests.test_gpu_tree_commit import caches_of, case
from tests.tree_util import i32

pytestmark = pytest.mark.gpu


def arguments(c):
    return [i32(c[k]) for k in ("parents", "tokens", "sampled", "offsets", "kv_lengths", "table")]


def moved(c, caches):
    """The caches with the accepted paths' rows moved, by the host oracle."""
    want = O.commit(c["parents"], c["tokens"], c["sampled"], c["offsets"], c["kv_lengths"], c["limit"], c["eos"],
                    c["table"].shape[1], c["page"])
    out = []
    for old in caches:
        now = old.clone()
        for r, w in enumerate(want):
            ctx = int(c["kv_lengths"][r] - (c["offsets"][r + 1] - c["offsets"][r]))
            for j, node in enumerate(w["path"]):
                (sb, so), (db, do) = (divmod(ctx + i, c["page"]) for i in (node, j))
                now[int(c["table"][r, db]), do] = old[int(c["table"][r, sb]), so]
        out.append(now)
    return out


def test_the_host_does_not_wait():
    rng = np.random.default_rng(1)
    c = case(rng, [20] * 6, 8)
    caches, args, limit = caches_of(rng, c, 5, 2, 64), arguments(c), i32(c["limit"])
    tree.commit_tree(*args, [t.clone() for t in caches], output_limit=limit)  # memory and code are there
    want = moved(c, caches)
    a = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
    b = torch.empty_like(a)
    torch.cuda.synchronize()
    for _ in range(200):  # about 0.2 s of work
        torch.mm(a, a, out=b)
    ahead = torch.cuda.Event()
    ahead.record()
    tree.commit_tree(*args, caches, output_limit=limit)
    assert not ahead.query()  # still at the work in front of the call
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(caches, want))


@pytest.mark.parametrize("count", [1, 128, 129, 300])
def test_many_caches_with_the_launch(count):
    """More caches than one launch's arguments hold."""
    rng = np.random.default_rng(count)
    c = case(rng, [9, 30, 2], 4)
    caches, args = caches_of(rng, c, count, 2, 16), arguments(c)
    again = [t.clone() for t in caches]
    want = moved(c, caches)
    a = tree.commit_tree(*args, caches, output_limit=i32(c["limit"]))
    b = tree.PreparedCommit(*args, again, output_limit=i32(c["limit"])).launch()
    assert all(torch.equal(x, y) for x, y in zip(caches, want)) and all(torch.equal(x, y) for x, y in zip(again, want))
    assert all(torch.equal(x, y) for x, y in zip(vars(a).values(), vars(b).values()))


def test_the_call_in_a_graph():
    rng = np.random.default_rng(2)
    c = case(rng, [20] * 6, 8)
    caches, args, limit = caches_of(rng, c, 140, 2, 64), arguments(c), i32(c["limit"])
    start = [t.clone() for t in caches]
    tree.commit_tree(*args, caches, output_limit=limit)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = tree.commit_tree(*args, caches, output_limit=limit)
    for turn in range(4):
        c["sampled"] = rng.integers(0, 2, len(c["sampled"]))
        args[2].copy_(i32(c["sampled"]))
        for t, s in zip(caches, start):
            t.copy_(s)
        want = moved(c, start)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(caches, want)), turn
        eager = tree.commit_tree(*args, [t.clone() for t in start], output_limit=limit)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(vars(got).values(), vars(eager).values())), turn


@pytest.mark.parametrize("upload", [False, True])
def test_a_cache_listed_twice_is_moved_once(upload):
    """Keys that are also the values: moved twice, a path's rows would move on."""
    rng = np.random.default_rng(4)
    c = case(rng, [40] * 5, 8)
    for r in range(5):  # every second node of a chain's siblings is kept
        c["parents"][40 * r:40 * r + 40] = [-1] + [2 * ((i - 1) // 2) for i in range(1, 40)]
    c["tokens"][:], c["sampled"][:], c["limit"][:] = np.arange(200) % 2, 0, 64
    caches, args = caches_of(rng, c, 3, 2, 64), arguments(c)
    want = moved(c, caches)
    assert not all(torch.equal(x, y) for x, y in zip(caches, want))
    often = 50 * caches  # more than one launch's, where the addresses go with it
    tree.PreparedCommit(*args, often, output_limit=i32(c["limit"]), upload=upload).launch()
    assert all(torch.equal(x, y) for x, y in zip(caches, want))
