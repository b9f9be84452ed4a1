"""The host oracle's plan and commit one after the other, without a GPU: what
a step refuses goes on from where it was."""
import numpy as np

from oracle import tree_oracle as O


def test_a_request_that_lacks_pages_goes_on_later():
    lengths, held, pending = np.array([40, 40, 40]), np.array([3, 3, 3]), np.array([7, 8, 9])
    table = np.full((3, 6), -1, np.int32)
    table[:, :3] = np.arange(9).reshape(3, 3)
    pool, state = np.array([9, -1, -1, -1]), np.array([0, 1])
    added = np.array([9, 9, 9])  # 49 tokens: a fourth page of 16
    parents = np.tile(np.arange(-1, 8), 3)
    plan = O.plan(lengths, added, table, held, pool, state, 10, 16, 27, parents)
    assert list(plan["status"]) == [O.OK, O.E_BLOCKS, O.E_BLOCKS]
    args = (parents, np.full(27, 5), np.full(27, 5), plan["offsets"], plan["kv_lengths"], [64] * 3, [set()] * 3, 6, 16)
    lost = O.commit(*args)
    assert [d["length"] for d in lost] == [49, 0, 0]  # what a loop must not go on with
    kept = O.commit(*args, before=(lengths, pending, plan["status"]))
    assert [d["length"] for d in kept] == [49, 40, 40]
    assert [d["pending"] for d in kept] == [5, 8, 9]
    assert [d["status"] for d in kept] == [O.OK, O.E_BLOCKS, O.E_BLOCKS]
    assert [len(d["ids"]) for d in kept] == [9, 0, 0] and not kept[1]["path"]


def test_requests_without_new_tokens_keep_their_pending_token():
    kv, none = np.array([12, 0]), np.zeros(3, int)
    d = O.commit([], [], [], none, kv, [0, 0], [set()] * 2, 4, 16, before=(np.array([12, 30]), [5, 6], [O.OK, O.OK]))
    assert [x["pending"] for x in d] == [5, 6] and [x["length"] for x in d] == [12, 0]
    assert [x["status"] for x in d] == [O.OK, O.OK]
