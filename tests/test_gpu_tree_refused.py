"""Steps that refuse some of their requests: plan_blocks, tree_attention and
commit_tree together, against the host oracle, and the loop that goes on."""
import ctypes

import numpy as np
import pytest
import torch

from deepseekrpc_amd import _native as N
from deepseekrpc_amd import tree
from examples import tree_decode
from oracle import tree_oracle as O
from tests.tree_util import i32, random_table, random_tree

pytestmark = pytest.mark.gpu
PAGE = 8


def state_of(rng, lengths, blocks, free):
    """Requests of these lengths with just the pages they need; a pool of ``free`` others."""
    held = -(-lengths // PAGE)
    table, rest = random_table(rng, list(held), blocks, spare=12)
    pool = np.full(blocks, -1, np.int32)
    pool[:free] = rest[:free]
    return dict(lengths=lengths, held=held, table=table, pool=pool, state=np.array([0, free]))


def step(rng, s, added, pending, blocks, capacity=None, parents=None, sampled=None):
    """One step on the device beside the oracle; what they agree on."""
    R = len(added)
    capacity = capacity or max(1, int(added.clip(0).sum()))
    if parents is None:
        parents = np.concatenate([np.array(random_tree(rng, int(max(0, a))), np.int64) for a in added])
    parents = np.concatenate([parents, np.full(capacity, -1)])[:capacity]
    tokens = rng.integers(0, 2, capacity)
    sampled = rng.integers(0, 2, capacity) if sampled is None else sampled
    limit = np.full(R, 64)
    want_plan = O.plan(**{k: s[k] for k in ("lengths", "table", "held", "pool", "state")}, added=added, blocks=blocks,
                       page=PAGE, capacity=capacity, parents=parents)
    dev = {k: i32(v) for k, v in s.items()}
    plan = tree.plan_blocks(dev["lengths"], i32(added), dev["table"], dev["held"], dev["pool"], dev["state"],
                            blocks=blocks, page=PAGE, capacity=capacity, parents=i32(parents))
    q, cache = torch.randn(capacity, 2, 64, device="cuda").half(), torch.randn(blocks, PAGE, 1, 64, device="cuda").half()
    att = tree.tree_attention(q, cache, cache, plan.table, plan.offsets, plan.kv_lengths, visible=plan.visible)
    before = cache.clone()
    done = tree.commit_tree(i32(parents), i32(tokens), i32(sampled), plan.offsets, plan.kv_lengths, plan.table, [cache],
                            output_limit=i32(limit), lengths=dev["lengths"], pending=i32(pending),
                            plan_status=plan.status)
    want = O.commit(parents, tokens, sampled, want_plan["offsets"], want_plan["kv_lengths"], limit, [set()] * R,
                    s["table"].shape[1], PAGE, before=(s["lengths"], pending, want_plan["status"]))
    np.testing.assert_array_equal(plan.status.cpu().numpy(), want_plan["status"])
    for key, of in (("lengths", "length"), ("pending", "pending"), ("stop", "stop"), ("status", "status")):
        assert getattr(done, key).tolist() == [w[of] for w in want], key
    assert done.accepted.tolist() == [len(w["path"]) for w in want]
    assert done.count.tolist() == [len(w["ids"]) for w in want]
    for r in np.flatnonzero(want_plan["status"]):
        lo, hi = want_plan["offsets"][r:r + 2]
        assert not att.out[lo:hi].any()
        ids = [int(b) for b in s["table"][r, :s["held"][r]] if 0 <= b < blocks]
        assert torch.equal(cache[ids], before[ids])  # its cached tokens stand where they were
    new = dict(lengths=done.lengths.cpu().numpy().astype(np.int64), held=dev["held"].cpu().numpy(),
               table=dev["table"].cpu().numpy(), pool=dev["pool"].cpu().numpy(), state=dev["state"].cpu().numpy())
    return new, done.pending.cpu().numpy(), want_plan["status"], want


@pytest.mark.parametrize("R", [4, 40])
def test_a_short_pool_for_a_step(R):
    rng = np.random.default_rng(R)
    lengths, blocks = rng.integers(1, 60, R), 20 * R
    s = state_of(rng, lengths, blocks, R // 2)
    pending, added = rng.integers(0, 100, R), np.full(R, 2 * PAGE)
    after, waiting, status, _ = step(rng, s, added, pending, blocks)
    short = status == O.E_BLOCKS
    assert short.any() and not short.all() and not status[~short].any()
    assert (after["lengths"][short] == lengths[short]).all() and (waiting[short] == pending[short]).all()
    # Pages come back: everyone is served from where they were.
    owned = np.concatenate([after["table"][r, :after["held"][r]] for r in range(R)])
    rest = np.setdiff1d(np.arange(blocks), owned)
    after["pool"][:len(rest)], after["state"] = rest, np.array([0, len(rest)])
    later, _, status, want = step(rng, after, added, waiting.clip(0), blocks)
    assert not status.any()
    assert (later["lengths"] == after["lengths"] + [len(w["path"]) for w in want]).all()


def test_token_arrays_too_short_malformed_trees_and_bad_pages():
    rng = np.random.default_rng(3)
    lengths, blocks = rng.integers(1, 40, 6), 100
    s = state_of(rng, lengths, blocks, 60)
    pending, added = np.arange(50, 56), np.array([9, 0, 17, 9, 9, 9])
    after, waiting, status, _ = step(rng, s, added, pending, blocks, capacity=30)  # 26 fit
    assert list(status) == [0, 0, 0, O.E_CAPACITY, O.E_CAPACITY, O.E_CAPACITY]
    kept = status != 0
    kept[1] = True  # no new tokens
    assert (after["lengths"][kept] == lengths[kept]).all() and (waiting[kept] == pending[kept]).all()

    s = state_of(rng, lengths, blocks, 60)
    s["table"][3, (lengths[3] - 1) // PAGE] = blocks  # where the new tokens go on
    s["lengths"][3] -= lengths[3] % PAGE == 0
    parents = np.concatenate([np.array(random_tree(rng, int(a)), np.int64) for a in added])
    parents[2] = 5
    after, waiting, status, _ = step(rng, s, added, pending, blocks, parents=parents)
    assert list(status) == [O.E_TREE, 0, 0, O.E_BLOCK, 0, 0]
    assert (after["lengths"][[0, 1, 3]] == s["lengths"][[0, 1, 3]]).all()
    assert (waiting[[0, 1, 3]] == pending[[0, 1, 3]]).all()


def test_no_token_drawn_and_ended_requests():
    rng = np.random.default_rng(5)
    lengths, blocks = np.array([20, 33, 0, 7]), 60
    s = state_of(rng, lengths, blocks, 30)
    added = np.array([5, -1, 4, 3])
    sampled = np.zeros(12, np.int64)
    sampled[0] = -1  # the sampler refused the root's row
    after, waiting, status, want = step(rng, s, added, np.array([3, 4, 5, 6]), blocks, sampled=sampled)
    assert not status.any() and [w["status"] for w in want] == [O.E_TOKEN, 0, 0, 0]
    assert after["lengths"][0] == 20 and waiting[0] == 3 and after["lengths"][1] == 0 and after["held"][1] == 0


@pytest.mark.parametrize("page,missing", [(16, 3), (16, 4)])
def test_greedy_output_is_the_same_with_a_short_pool(page, missing):
    model = tree_decode.Model()
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, 512, n).tolist() for n in (3, 1, 70, 18, 33)]
    roomy = tree_decode.generate(model, prompts, 40, page=page)
    short = tree_decode.generate(model, prompts, 40, page=page, missing=missing)
    assert [o.ids for o in short] == [o.ids for o in roomy]
    assert sum(o.waits for o in short) > 0 and sum(o.waits for o in roomy) == 0


def test_refused_arguments():
    """The state before the step comes whole, and in no output."""
    one, two = i32([3]), i32([3, 4])
    good = (i32([-1]), one, one, i32([0, 1]), one, i32([[0]]), [])
    kw = dict(output_limit=one, page=PAGE, blocks=4)
    res = tree.commit_tree(*good, **kw, lengths=i32([2]), pending=one, plan_status=i32([0]))
    assert res.lengths.tolist() == [3]
    for bad in (dict(lengths=one), dict(lengths=one, pending=one), dict(pending=one, plan_status=one),
                dict(lengths=one, pending=one, plan_status=two), dict(lengths=one.long(), pending=one, plan_status=one),
                dict(lengths=one, pending=one.cpu(), plan_status=one)):
        with pytest.raises((TypeError, ValueError)):
            tree.commit_tree(*good, **kw, **bad)
    call = tree.PreparedCommit(*good, **kw, lengths=i32([2]), pending=one, plan_status=i32([0]))
    for field, value in (("lengths_in", call.args.lengths), ("pending_in", call.args.pending),
                         ("plan_status", call.args.status), ("lengths_in", None), ("plan_status", None)):
        keep = getattr(call.args, field)
        setattr(call.args, field, value)
        assert N.load().dsr_commit_tree(ctypes.byref(call.args), None) == -1, field
        setattr(call.args, field, keep)
