"""dsr_select_beams against the host oracle: the same rows and tokens, scores
within the rounding of float64."""
import math

import numpy as np
import pytest
import torch

from deepseekrpc_amd import branches
from oracle import branch_oracle as O
from tests.tree_util import DTYPES, i32

pytestmark = pytest.mark.gpu


def rows_of(rng, rows, V, dtype, ld=None, offset=0):
    """Logits of the type, as a view of wider rows if asked, and what they are on the host."""
    ld = ld or V
    buf = torch.zeros(rows * ld + offset, dtype=DTYPES[dtype], device="cuda")
    t = buf[offset:].view(rows, ld)[:, :V]
    t.copy_(torch.from_numpy((rng.standard_normal((rows, V)) * 3).astype(np.float32)))
    return t


def check(logits, scores, offsets, keep, finished=None):
    s = torch.tensor(scores, dtype=torch.float64, device="cuda")
    f = None if finished is None else i32(finished)
    res = branches.select_beams(logits, s, i32(offsets), keep=keep, finished=f)
    groups, status = O.select(logits.double().cpu().numpy(), scores, offsets, keep, finished)
    assert res.status.tolist() == status
    V = logits.shape[1]
    for g, (parents, tokens, best) in enumerate(groups):
        assert res.parents[g].tolist() == parents, g
        assert res.tokens[g].tolist() == tokens, g
        for got, want in zip(res.scores[g].tolist(), best):
            # The sum of V exponentials of 2^-51 each, a table's or a polynomial's
            # rounding of 8 2^-53, then 40 additions in a row (a thread's 32, lanes,
            # waves, slices), the logarithm's last bit, three additions of at most |score| + 40 + log V.
            bound = 2.0**-53 * (60 + V / 4096 + 8 * (abs(want) + 40 + math.log(V))) if math.isfinite(want) else 0
            assert got == want or abs(got - want) <= bound, (g, got, want)
    return res


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("groups,beams,V,keep", [
    (1, 1, 1, 1), (1, 1, 1, 64), (3, 4, 7, 5), (2, 3, 100, 64), (1, 4, 8191, 8), (1, 4, 8192, 8), (2, 2, 8193, 8),
    (5, 4, 32000, 4), (2, 8, 129280, 16), (1, 16, 50257, 32), (2, 2, 129280, 64)])
def test_matches_the_oracle(groups, beams, V, keep, dtype):
    rng = np.random.default_rng([groups, beams, V, keep])
    scores = -20 * rng.random(groups * beams)
    check(rows_of(rng, groups * beams, V, dtype), scores, np.arange(groups + 1) * beams, keep)


@pytest.mark.parametrize("ld,offset", [(1000, 0), (1001, 0), (1008, 3), (1008, 8)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_of_any_alignment(ld, offset, dtype):
    rng = np.random.default_rng([ld, offset])
    check(rows_of(rng, 6, 997, dtype, ld, offset), -rng.random(6), [0, 2, 6], 6)


def test_ragged_empty_and_partial_groups():
    """Groups of no rows, of different ones, of rows that others have too, and rows of none."""
    rng = np.random.default_rng(1)
    x, s = rows_of(rng, 9, 333, "bf16"), -rng.random(9)
    check(x, s, [1, 1, 4, 8], 5)
    check(x, s, [0], 5)
    check(x, s, [0, 6, 3, 9], 5)
    check(x, s, [-4, 2, 700], 5)  # bounds are held to the rows


def test_ended_dead_and_masked_rows():
    rng = np.random.default_rng(2)
    x = rows_of(rng, 10, 500, "bf16")
    x[1] = -math.inf
    x[2, 1:] = -math.inf
    x[3, ::2] = -math.inf
    x[5] = math.nan  # ended: never read
    x[6] = torch.finfo(torch.bfloat16).min
    scores = [-1.0, -0.5, -0.25, -2.0, -math.inf, -0.75, -3.0, -1.5, -math.inf, -1.25]
    finished = [0, 0, 0, 0, 0, 1, 0, -7, 1, 0]
    for offsets in ([0, 10], [0, 5, 10], [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10]):
        for keep in (1, 4, 64):
            check(x, scores, offsets, keep, finished)


def test_rows_that_are_not_numbers_offer_nothing():
    rng = np.random.default_rng(3)
    for dtype in ("bf16", "f16", "f32"):
        x = rows_of(rng, 7, 9000, dtype)
        x[1, 8999] = math.nan
        x[2, 0] = math.inf
        x[3, 17], x[3, 18] = math.nan, -math.inf
        check(x, [-1.0, -1, -1, -1, math.nan, math.inf, -1], [0, 4, 7], 8)
        check(x, [-1.0, -1, -1, -1, math.nan, math.inf, -1], [0, 7], 8, [0, 0, 0, 0, 1, 1, 1])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_equal_offers_go_to_the_lowest_row_and_token(dtype):
    rng = np.random.default_rng(4)
    x = rows_of(rng, 4, 20000, dtype)
    x[:] = 0  # every offer the same
    check(x, [-1.0] * 4, [0, 4], 64)
    x[:, 77] = -0.0
    check(x, [-1.0] * 4, [0, 2, 4], 33)
    x[:] = torch.from_numpy(rng.integers(-3, 4, (4, 20000)).astype(np.float32))  # thousands of equals
    x[2] = x[0]
    check(x, [-1.0, -1.5, -1.0, -2.0], [0, 4], 64)
    # Ascending: the last are best.
    y = torch.arange(20000, device="cuda").float().expand(4, -1).div(64).to(DTYPES[dtype])
    check(y, [-1.0, -1.5, -1.25, -2.0], [0, 4], 64)
    z = y.flip(1).contiguous()
    check(z, [-1.0, -1.5, -1.25, -2.0], [0, 4], 64)


def test_many_rows_of_one_group():
    rng = np.random.default_rng(5)
    check(rows_of(rng, 1500, 40, "f32"), -20 * rng.random(1500), [0, 1500], 64)
    check(rows_of(rng, 700, 30, "bf16"), -20 * rng.random(700), np.arange(701), 3)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,V,ld,offset", [
    (512, 16384, 16384, 0), (512, 16389, 16392, 0), (512, 4099, 4099, 0), (515, 2048, 2056, 8),
    (256, 9001, 9001, 0), (256, 8200, 8200, 0), (256, 12289, 12296, 0), (300, 8193, 8200, 1)])
def test_many_logits_a_thread(rows, V, ld, offset, dtype):
    """Rows enough for 64 or 32 logits a thread.  64 additions in a row in place of
    32 are 32 roundings more, of which check()'s bound has 5 x 40 to spare."""
    rng = np.random.default_rng([rows, V, ld, offset])
    offsets = [rows - 20, rows - 17, rows - 8, rows - 8, rows]
    x = rows_of(rng, rows, V, dtype, ld, offset)
    x[-18, V // 2:] = -math.inf
    x[-16, : V - 1] = -math.inf
    x[-15, V - 1] = math.nan
    finished = np.arange(rows) % 24 != rows % 24  # the others are there for their number
    finished[-20:] = rng.random(20) < 0.1
    check(x, -20 * rng.random(rows), offsets, 9, finished.astype(np.int32).tolist())


def test_far_scores_and_logits():
    """Scores a long output's, logits far apart: nothing is lost in between."""
    rng = np.random.default_rng(6)
    x = rows_of(rng, 4, 3000, "f32")
    x *= 300
    check(x, [-1e5, -1e5 - 1e-9, -2e5, -1e5 + 1e-9], [0, 4], 16)
    x[1] = 3e38
    x[2] = -3e38
    check(x, [-10.0] * 4, [0, 4], 16)
    x[1, 5:] = 1e38  # a step of float32 here is far more than the exponential's range
    x[3] += 1e12
    check(x, [-10.0, -1e38, -10, -10], [0, 1, 2, 3, 4], 16)


def test_a_prepared_call_in_a_graph_and_on_another_stream():
    rng = np.random.default_rng(7)
    x, s = rows_of(rng, 8, 9000, "bf16"), torch.tensor(-rng.random(8), device="cuda")
    p = branches.PreparedBeams(x, s, i32([0, 4, 8]), keep=8)
    p.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = p.launch()
    for turn in range(3):
        x.copy_(rows_of(rng, 8, 9000, "bf16"))
        graph.replay()
        torch.cuda.synchronize()
        here = [t.clone() for t in (got.parents, got.tokens, got.scores, got.status)]
        check(x, s.tolist(), [0, 4, 8], 8)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = branches.select_beams(x, s, i32([0, 4, 8]), keep=8)
        torch.cuda.synchronize()
        for a, b in zip(here, (other.parents, other.tokens, other.scores, other.status)):
            assert torch.equal(a, b), turn


def test_refusals():
    x, s, o = torch.zeros(4, 10, device="cuda"), torch.zeros(4, dtype=torch.float64, device="cuda"), i32([0, 4])
    call = lambda *a, **k: branches.select_beams(*a, **{"keep": 2, **k})  # noqa: E731
    with pytest.raises(TypeError):
        call(x.cpu(), s, o)
    for bad in (lambda: call(x.double(), s, o), lambda: call(x, s.float(), o), lambda: call(x, s[:3], o),
                lambda: call(x.t(), s, o), lambda: call(x, s, o.long()), lambda: call(x, s, o, keep=0),
                lambda: call(x, s, o, keep=65), lambda: call(x, s, o, keep=2.0), lambda: call(x, s, o[:0]),
                lambda: call(x[:, :0], s, o), lambda: call(x, s, o, finished=s),
                lambda: call(x.clone().requires_grad_(), s, o), lambda: call(x, s, o, out=dict(other=s)),
                lambda: call(x, s, o, out=dict(scores=s.view(1, 4)[:, :2])),
                lambda: call(x, s, o, out=dict(tokens=i32([[1, 2, 3]])))):
        with pytest.raises(ValueError):
            bad()
