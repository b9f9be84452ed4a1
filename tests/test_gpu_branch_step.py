"""The operators of decoding with several branches one after the other, as a
beam search calls them: every result against the host oracles, and what each row
reads through its table against the tokens that it has."""
import types

import numpy as np
import pytest
import torch

from deepseekrpc_amd import branches, tree
from examples import beam_decode
from oracle import branch_oracle as O
from oracle import tree_oracle as T
from tests.tree_exact import check
from tests.tree_util import i32

pytestmark = pytest.mark.gpu


def host(t):
    return t.cpu().numpy()


@pytest.mark.parametrize("page,dim,beams", [(8, 64, 4), (16, 128, 3), (1, 64, 2)])
def test_steps_of_beams(page, dim, beams):
    rng = np.random.default_rng([page, dim])
    prompts, heads, kv, V, width, blocks = [37, 5, 64], 8, 2, 500, 40 if page > 1 else 120, 400
    R, dev = len(prompts), "cuda"
    k_cache = torch.zeros(blocks, page, kv, dim, dtype=torch.bfloat16, device=dev)
    v_cache = torch.zeros_like(k_cache)
    pool, state = tree.page_pool(blocks)
    shared = torch.zeros(blocks, dtype=torch.int32, device=dev)
    table = torch.full((R, width), -1, dtype=torch.int32, device=dev)
    held, lengths, added = i32([0] * R), i32([0] * R), np.array(prompts)
    freqs, _ = tree.rotary_frequencies(dim)
    rows, scores, offsets, finished = R, np.zeros(R), np.arange(R + 1), np.zeros(R, np.int32)
    told = [([], []) for _ in range(R)]  # what each row's keys and values were
    groups, prefix = i32([0] * (R + 1)), i32([0] * R)

    def normal(*s):
        return torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(dev, torch.bfloat16)

    for step in range(14):
        n = int(added.clip(0).sum())
        plan = tree.plan_blocks(lengths, i32(added), table, held, pool, state, blocks=blocks, page=page, capacity=n + 2)
        assert not plan.status.any()
        q, k, v = normal(n + 2, heads, dim), normal(n + 2, kv, dim), normal(n + 2, kv, dim)
        q = tree.rotary(q, k, plan.positions, freqs, v=v, slots=plan.slots, k_cache=k_cache, v_cache=v_cache).q
        slots, off = host(plan.slots), host(plan.offsets)
        flat_k, flat_v = k_cache.view(-1, kv, dim), v_cache.view(-1, kv, dim)
        for r in range(rows):
            at = torch.from_numpy(slots[off[r]:off[r + 1]].astype(np.int64)).to(dev)
            told[r] = (told[r][0] + list(flat_k[at]), told[r][1] + list(flat_v[at]))
        if step == 0:
            res = tree.tree_attention(q, k_cache, v_cache, plan.table, plan.offsets, plan.kv_lengths, lse=True)
        else:
            res = branches.prefix_attention(q, k_cache, v_cache, plan.table, plan.offsets, plan.kv_lengths, groups,
                                            prefix, lse=True)
        assert not res.status.any()
        if step in (0, 1, 5, 13):
            check(types.SimpleNamespace(page=page, q=q, k=k_cache, v=v_cache, table=host(plan.table), offsets=off,
                                        kv_lengths=host(plan.kv_lengths), visible=None), res, "bf16")
        lengths = plan.kv_lengths
        # The next step's rows.
        logits = normal(rows, V) * 4
        best = branches.select_beams(logits, torch.from_numpy(scores).to(dev), i32(offsets), keep=beams,
                                     finished=i32(finished))
        want, status = O.select(logits.double().cpu().numpy(), scores, offsets, beams, finished)
        assert not any(status)
        assert host(best.parents).tolist() == [p for p, _, _ in want]
        assert host(best.tokens).tolist() == [t for _, t, _ in want]
        parents, tokens = host(best.parents).ravel(), host(best.tokens).ravel()
        want = O.fork(host(lengths), parents, host(table), host(held), host(shared), host(pool), host(state), blocks,
                      page)
        fork = branches.fork_pages(lengths, best.parents.flatten(), table, held, shared, pool, state,
                                   [k_cache, v_cache])
        for f in ("table", "held", "lengths", "shared", "pool", "state", "status", "source_status"):
            np.testing.assert_array_equal(host(getattr(fork, f)), want[f], err_msg=f)
        assert not any(want["status"])
        table, held, lengths = fork.table, fork.held, fork.lengths
        told = [(list(told[p][0]), list(told[p][1])) for p in parents]
        if step % 4 == 2:
            before = host(state)[1]
            c = branches.compact_pages(table, held, pool, state, [k_cache, v_cache], shared=shared)
            assert not c.status.any() and host(state)[1] == before and int(host(table).max()) < blocks - before
        rows, scores = R * beams, host(best.scores).ravel()
        finished = (finished[parents] != 0) | (tokens < 0) | (rng.random(rows) < 0.04)
        finished = finished.astype(np.int32)
        offsets = np.arange(R + 1) * beams
        groups, prefix = i32(offsets), i32([p // page * page for p in prompts])
        added = 1 - finished
        for r in range(rows):  # every row reads what its tokens wrote
            at = np.arange(host(lengths)[r])
            ids = torch.from_numpy(host(table)[r, at // page].astype(np.int64)).to(dev)
            in_page = torch.from_numpy(at % page).to(dev)
            assert torch.equal(k_cache[ids, in_page], torch.stack(told[r][0])), (step, r)
            assert torch.equal(v_cache[ids, in_page], torch.stack(told[r][1])), (step, r)
    end = branches.fork_pages(lengths, i32([-1] * rows), table, held, shared, pool, state, [], page=page, blocks=blocks)
    assert int(state[1]) == blocks and not shared.any() and not end.held.any()
    assert sorted(host(pool).tolist()) == list(range(blocks))


@pytest.mark.parametrize("page,every", [(16, 0), (4, 3), (1, 0)])
def test_the_example_runs_and_gives_every_page_back(page, every):
    model = beam_decode.Model()
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, 512, n).tolist() for n in (3, 1, 70, 18, 33)]
    out, free, blocks = beam_decode.search(model, prompts, 20, 4, page=page, eos=7, compact_every=every)
    assert free == blocks
    for found in out:
        assert 1 <= len(found) <= 4 and all(1 <= len(ids) <= 20 for ids, _ in found)
        scores = [s for _, s in found]
        assert scores == sorted(scores, reverse=True) and len({tuple(ids) for ids, _ in found}) == len(found)


def test_one_beam_is_greedy_decoding():
    """With one beam the best token is the likeliest, as sample_rows takes it at temperature 0."""
    rng = np.random.default_rng(1)
    from deepseekrpc_amd import batch
    logits = torch.from_numpy((rng.standard_normal((6, 5000)) * 3).astype(np.float32)).cuda().to(torch.bfloat16)
    best = branches.select_beams(logits, torch.zeros(6, dtype=torch.float64, device="cuda"), i32(np.arange(7)), keep=1)
    u = torch.zeros(6, dtype=torch.float64, device="cuda")
    greedy = batch.sample_rows(logits, [dict(temperature=0.0)] * 6, uniforms=u)
    assert torch.equal(best.tokens[:, 0], greedy.tokens)
