"""Page ids outside the cache: none of the request's tokens gets a slot, on
whatever page they would lie and in whatever part of the work they fall."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import tree
from oracle import tree_oracle as O
from tests.test_gpu_tree_plan import case, check
from tests.tree_util import i32

pytestmark = pytest.mark.gpu


def with_bad_pages(c, rng, requests, blocks):
    """The last touched page of some requests, held or from the pool, is outside."""
    fine = O.plan(**c)
    for r in requests:
        L, A, held = int(c["lengths"][r]), int(c["added"][r]), int(c["held"][r])
        if A <= 0:
            continue
        b = (L + A - 1) // c["page"]
        at = np.flatnonzero(c["pool"] == fine["table"][r, b]) if b >= held else []
        bad = int(rng.choice([-1, blocks, 2**31 - 1, -2**31]))
        if len(at):
            c["pool"][at[0]] = bad
        else:
            c["table"][r, b] = bad
    return c


@pytest.mark.parametrize("R,new_hi,context,page", [(1, 5, 40, 2), (3, 300, 40, 8), (40, 30, 100, 8), (700, 30, 100, 8),
                                                   (5, 5000, 300, 16), (2, 40_000, 5, 1), (300, 200, 2000, 64)])
@pytest.mark.parametrize("trees", [False, True])
@pytest.mark.parametrize("share", [0.05, 0.6])
def test_no_token_of_a_refused_request_has_a_slot(R, new_hi, context, page, trees, share):
    rng = np.random.default_rng([R, new_hi, page, trees])
    c = case(rng, R, min(new_hi, 64) if trees else new_hi, context, page, trees, ended=0.05, capacity_slack=70)
    hit = np.flatnonzero(rng.random(R) < share)
    hit = hit if len(hit) else np.array([R - 1])
    want = check(with_bad_pages(c, rng, hit, c["blocks"]))
    refused = want["status"] == O.E_BLOCK
    assert refused[hit[c["added"][hit] > 0]].all()
    mine = np.isin(want["owners"], np.flatnonzero(refused))
    assert (want["slots"][mine] == -1).all() and (want["positions"][mine] == 0).all()
    assert want["visible"] is None or not want["visible"][mine].any()


def test_bad_pages_that_the_step_does_not_touch():
    """Ids behind the touched pages, of full pages before them and of requests
    without tokens refuse nobody."""
    rng = np.random.default_rng(8)
    c = case(rng, 60, 100, 300, 8, False, ended=0.0)
    c["added"][::7] = 0
    c["capacity"] = int(c["added"].sum())
    for r in range(60):
        first, end = c["lengths"][r] // 8, -(-(c["lengths"][r] + c["added"][r]) // 8)
        c["table"][r, :first if c["added"][r] else None] = c["blocks"] + 3
        c["table"][r, max(end, c["held"][r]):] = -9
    used = c["state"][1] // 2
    want = O.plan(**c)
    used = int((want["held"] - c["held"]).sum())
    c["pool"][(c["state"][0] + np.arange(used, c["state"][1])) % len(c["pool"])] = -3  # not taken this time
    want = check(c)
    assert not want["status"].any()


@pytest.mark.parametrize("R,new_hi", [(16384, 1), (9000, 9), (2000, 70)])
@pytest.mark.parametrize("in_place", [True, False])
def test_pages_held_and_pool_replaced_in_place(R, new_hi, in_place):
    """The pages are looked through while the scan settles what is held and
    free: in many requests and in place, bad pages are found all the same."""
    rng = np.random.default_rng([R, new_hi])
    c = case(rng, R, new_hi, 40, 4, False, ended=0.02)
    hit = rng.choice(R, 12, replace=False)
    c["added"][hit] = new_hi
    c["capacity"] = max(1, int(c["added"].clip(0).sum()))
    want = check(with_bad_pages(c, rng, hit, c["blocks"]), in_place)
    assert (want["status"][hit] == O.E_BLOCK).all()


def test_results_in_memory_that_is_still_read():
    """Lengths replaced by the plan's own lengths would move every later token."""
    lengths, added, held, state = i32([9, 20]), i32([3, 2]), i32([2, 3]), i32([0, 4])
    table, pool = i32([[0, 1, -1], [2, 3, 4]]), i32([5, 6, 7, 8])
    args, kw = (lengths, added, table, held, pool, state), dict(blocks=9, page=8, capacity=5)
    buffer = i32(np.zeros(40))
    good = [dict(held=held, state=state), dict(held=torch.empty_like(held)), dict(slots=buffer[:5], owners=buffer[5:10]),
            dict(slots=None, kv_lengths=buffer[:2])]
    for out in good:
        tree.PreparedPlan(*args, **kw, out=out)
    for out in (dict(kv_lengths=lengths), dict(kv_lengths=added), dict(status=lengths), dict(status=held),
                dict(held=lengths), dict(state=added), dict(offsets=pool[:3]), dict(kv_lengths=table[1, :2]),
                dict(slots=buffer[:5], owners=buffer[4:9]), dict(slots=buffer[:5], positions=buffer[:5])):
        with pytest.raises(ValueError, match="overlap"):
            tree.PreparedPlan(*args, **kw, out=out)
