"""The host oracle of forked and compacted pages against what the operators are
for, without a GPU: every row reads the tokens of the row that it continues."""
import numpy as np

from oracle import branch_oracle as O


def read(cache, row, length, page):
    return [int(cache[row[i // page], i % page]) for i in range(length)]


def moved(cache, copies):
    now = cache.copy()
    for a, b, n in copies:
        now[b, :n] = cache[a, :n]
    return now


def test_rows_read_what_their_sources_hold():
    rng = np.random.default_rng(1)
    page, blocks, width = 4, 60, 8
    cache = rng.integers(0, 1 << 30, (blocks, page))
    lengths, held = [10, 8, 0, 5], [4, 2, 0, 2]
    table = np.full((4, width), -1)
    perm = list(rng.permutation(blocks))
    shared = np.zeros(blocks, int)
    for r in range(4):
        table[r, :held[r]] = [perm.pop() for _ in range(held[r])]
    pool, state = np.full(blocks, -1), [17, len(perm)]
    pool[(17 + np.arange(len(perm))) % blocks] = perm
    for _ in range(30):
        parents = rng.integers(-1, len(lengths), 6)
        d = O.fork(lengths, parents, table, held, shared, pool, state, blocks, page)
        assert not any(d["status"]) and not any(d["source_status"])
        now = moved(cache, d["copies"])
        for r, p in enumerate(parents):
            if p >= 0:
                assert read(now, d["table"][r], d["lengths"][r], page) == read(cache, table[p], lengths[p], page)
        holders = np.zeros(blocks, int)
        for row, n in zip(d["table"], d["held"]):
            holders[row[:n]] += 1
        assert (np.maximum(holders - 1, 0) == d["shared"]).all()
        assert (holders > 0).sum() + d["state"][1] == blocks
        # Only full pages are shared.
        for row, n, length in zip(d["table"], d["held"], d["lengths"]):
            assert not d["shared"][row[length // page:n]].any()
        cache, lengths, held, table = now, d["lengths"], d["held"], d["table"]
        shared, pool, state = d["shared"], d["pool"], d["state"]
        c = O.compact(table, held, shared, pool, state, blocks, page)
        now = moved(cache, c["copies"])
        for old, new, n in zip(table, c["table"], lengths):
            assert read(now, new, n, page) == read(cache, old, n, page)
        assert sorted(set(c["table"][c["table"] >= 0])) == list(range(blocks - c["state"][1]))
        cache, table, shared, pool, state = now, c["table"], c["shared"], np.array(c["pool"]), c["state"]


def test_beams_of_one_step():
    logits = np.log(np.array([[0.5, 0.25, 0.25], [0.1, 0.1, 0.8]]))
    groups, status = O.select(logits, [0.0, -1.0], [0, 2], 4)
    parents, tokens, scores = groups[0]
    assert parents == [0, 1, 0, 0] and tokens == [0, 2, 1, 2] and status == [0, 0]
    np.testing.assert_allclose(scores, [np.log(0.5), np.log(0.8) - 1, np.log(0.25), np.log(0.25)], atol=1e-15)
    groups, _ = O.select(logits, [0.0, -1.0], [0, 2], 5, finished=[0, 1])
    assert groups[0][0] == [0, 1, 0, 0, -1] and groups[0][1] == [0, -1, 1, 2, -1]
