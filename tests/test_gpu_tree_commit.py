"""dsr_commit_tree against the host oracle: decisions and moved rows are equal."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import tree
from oracle import tree_oracle as O
from tests.tree_util import i32, random_table, random_tree

pytestmark = pytest.mark.gpu


def case(rng, new, page, vocab=2, context=60, limit=64):
    ctx = rng.integers(0, context + 1, len(new))
    kv = ctx + np.array(new)
    pages = [-(-int(x) // page) for x in kv]
    blocks = max(1, sum(pages)) + 1
    table, _ = random_table(rng, pages, blocks)
    n = sum(new)
    return dict(parents=np.concatenate([np.array(random_tree(rng, m), np.int64) for m in new]) if n else np.zeros(0, int),
                tokens=rng.integers(0, vocab, n), sampled=rng.integers(0, vocab, n),
                offsets=np.concatenate([[0], np.cumsum(new)]), kv_lengths=kv, table=table, page=page, blocks=blocks,
                limit=rng.integers(1, limit + 1, len(new)), eos=[set() for _ in new])


def check(c, caches):
    R, page = len(c["kv_lengths"]), c["page"]
    want = O.commit(c["parents"], c["tokens"], c["sampled"], c["offsets"], c["kv_lengths"], c["limit"], c["eos"],
                    c["table"].shape[1], page)
    eos_off = torch.tensor(np.concatenate([[0], np.cumsum([len(e) for e in c["eos"]])]), dtype=torch.int64).cuda()
    eos = i32([t for e in c["eos"] for t in sorted(e)])
    before = [t.clone() for t in caches]
    kw = dict(page=page, blocks=c["blocks"]) if not caches else {}
    res = tree.commit_tree(*(i32(c[k]) for k in ("parents", "tokens", "sampled", "offsets", "kv_lengths", "table")),
                           caches, output_limit=i32(c["limit"]), eos_offsets=eos_off, eos_ids=eos, **kw)
    pad = lambda x: x + [-1] * (64 - len(x))  # noqa: E731
    for r in range(R):
        w = want[r]
        got = {k: getattr(res, k)[r].tolist() for k in ("path", "ids", "accepted", "count", "pending", "stop",
                                                        "lengths", "status")}
        assert got == dict(path=pad(w["path"]), ids=pad(w["ids"]), accepted=len(w["path"]), count=len(w["ids"]),
                           pending=w["pending"], stop=w["stop"], lengths=w["length"], status=w["status"]), r
    for old, now in zip(before, caches):
        old = old.clone()
        new_rows = old.clone()
        for r, w in enumerate(want):
            ctx = int(c["kv_lengths"][r] - (c["offsets"][r + 1] - c["offsets"][r]))
            for j, node in enumerate(w["path"]):
                s, d = ctx + node, ctx + j
                new_rows[int(c["table"][r, d // page]), d % page] = old[int(c["table"][r, s // page]), s % page]
        assert torch.equal(now, new_rows)
    return want


def caches_of(rng, c, count, heads, dim, dtype=torch.bfloat16, by_head=False):
    shape = (c["blocks"], heads, c["page"], dim) if by_head else (c["blocks"], c["page"], heads, dim)
    out = [torch.from_numpy(rng.integers(-100, 100, shape).astype(np.float32)).cuda().to(dtype) for _ in range(count)]
    return [t.transpose(1, 2) for t in out] if by_head else out


@pytest.mark.parametrize("new,page", [([1], 16), ([2], 1), ([64, 64, 64], 16), ([5, 0, 17, 33], 8), ([64] * 9, 64),
                                      ([30] * 40, 4)])
@pytest.mark.parametrize("count,heads,dim,by_head", [(1, 1, 8, False), (3, 2, 64, True), (17, 8, 128, False)])
def test_paths_and_rows(new, page, count, heads, dim, by_head):
    rng = np.random.default_rng([sum(new), page, count])
    c = case(rng, new, page)
    c["eos"] = [{1} if r % 3 == 1 else {5, 0} if r % 3 == 2 else set() for r in range(len(new))]
    check(c, caches_of(rng, c, count, heads, dim, by_head=by_head))


def test_a_whole_chain_and_siblings():
    rng = np.random.default_rng(2)
    c = case(rng, [64, 8, 8], 16, limit=100)
    c["limit"][:] = 100
    c["tokens"][:] = 7
    c["sampled"][:] = 7
    c["parents"][:64] = np.arange(-1, 63)          # a chain, all accepted: nothing moves
    c["parents"][64:72] = [-1, 0, 0, 0, 1, 2, 3, 3]  # equal siblings: the first
    c["parents"][72:80] = [-1, -1, 0, 1, 2, -1, 4, 4]  # other roots are never reached
    want = check(c, caches_of(rng, c, 2, 2, 16, torch.float32))
    assert want[0]["path"] == list(range(64)) and want[1]["path"] == [0, 1, 4] and want[2]["path"] == [0, 2, 4, 6]


@pytest.mark.parametrize("limit,eos,stop,pending", [(3, set(), 2, -1), (64, {7}, 1, -1), (1, set(), 2, -1)])
def test_stops_at_an_accepted_draft(limit, eos, stop, pending):
    rng = np.random.default_rng(3)
    c = case(rng, [10], 8)
    c["parents"][:] = np.arange(-1, 9)
    c["tokens"][:] = 7
    c["sampled"][:] = 7
    c["limit"][:], c["eos"] = limit, [eos]
    want = check(c, [])
    assert want[0]["stop"] == stop and want[0]["pending"] == pending
    c["tokens"][:] = 8                              # the pending token itself stops
    want = check(c, [])
    assert want[0]["path"] == [0] and want[0]["pending"] == 7


def test_statuses():
    rng = np.random.default_rng(4)
    c = case(rng, [6, 6, 65, 6, 6, 6], 8)
    c["parents"][1] = 3
    c["kv_lengths"][1] = 2
    c["limit"][3] = 0
    c["sampled"][c["offsets"][4]] = -1
    c["kv_lengths"][5] = c["table"].shape[1] * 8 + 1
    want = check(c, caches_of(rng, c, 2, 1, 8))
    assert [w["status"] for w in want] == [O.E_TREE, O.E_LENGTH, O.E_TREE, O.E_LENGTH, O.E_TOKEN, O.E_LENGTH]
    # A page id outside the cache: nothing is accepted.
    c = case(rng, [6, 6], 1, context=0)
    caches = caches_of(rng, c, 2, 1, 8)
    before = [t.clone() for t in caches]
    c["table"][0, 0] = c["blocks"]
    res = tree.commit_tree(*(i32(c[k]) for k in ("parents", "tokens", "sampled", "offsets", "kv_lengths", "table")),
                           caches, output_limit=i32([64, 64]))
    assert res.status.tolist() == [O.E_BLOCK, 0] and res.accepted[0] == 0 and (res.path[0] == -1).all()
    row = int(c["table"][1, 0])
    assert all(torch.equal(a[row], b[row]) for a, b in zip(caches, before))


def test_refused_arguments():
    rng = np.random.default_rng(5)
    c = case(rng, [4], 8)
    good = [i32(c[k]) for k in ("parents", "tokens", "sampled", "offsets", "kv_lengths", "table")]
    caches, lim = caches_of(rng, c, 2, 2, 16), i32([5])
    tree.commit_tree(*good, caches, output_limit=lim)
    for i, bad in ((0, good[0].long()), (1, good[1][:2]), (2, good[2].cpu()), (3, good[3][:1]), (4, good[4].float()),
                   (5, good[5].long())):
        with pytest.raises((TypeError, ValueError)):
            tree.commit_tree(*good[:i], bad, *good[i + 1:], caches, output_limit=lim)
    odd = torch.zeros(c["blocks"], 8, 2, 12, device="cuda", dtype=torch.bfloat16)
    for kw in (dict(caches=[]), dict(caches=[caches[0], caches[1].float()]), dict(caches=[odd]),
               dict(caches=[caches[0], caches[1][:, :, :1]]), dict(output_limit=lim.long()),
               dict(eos_ids=i32([1])), dict(caches=[c.cpu() for c in caches])):
        with pytest.raises((TypeError, ValueError)):
            tree.commit_tree(*good, **dict(dict(caches=caches, output_limit=lim), **kw))
    z = i32([])
    none = tree.commit_tree(z, z, z, i32([0]), z, torch.empty(0, 1, dtype=torch.int32, device="cuda"), caches,
                            output_limit=z)
    assert none.path.shape == (0, 64)
