"""dsr_prefix_attention against float64 attention of each request over its own
table row, row by row, within the bound of tests/tree_exact."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import branches, tree
from tests.branch_util import PrefixStep, far_apart
from tests.tree_exact import check
from tests.tree_util import i32

pytestmark = pytest.mark.gpu


def run(step, dtype, scale=None, **kw):
    args, vis = step.prefix_args()
    res = branches.prefix_attention(*args, visible=vis, scale=scale, lse=True, **kw)
    check(step, res, dtype, scale)
    return res


SHAPES = [  # family, prefixes, new, own, heads, kv, dim, page, alone
    (1, [16], [1], [0], 1, 1, 8, 16, 0),
    (2, [32], [1, 1], [0, 5], 4, 4, 64, 16, 0),
    (4, [96, 33], [1] * 8, [3, 0, 1, 70, 2, 2, 2, 9], 8, 2, 128, 1, 0),
    (3, [160], [1, 2, 1, 4], [31, 1, 400, 6], 10, 2, 96, 32, 1),
    (8, [1000], [1] * 8, [5] * 8, 16, 1, 128, 8, 0),
    (2, [64, 0, 640], [5, 1, 9, 1, 1, 17], [0, 1, 2, 3, 4, 5], 6, 3, 72, 64, 0),
    (5, [500], [3, 0, 17, 1, 33], [0, 0, 100, 200, 1], 4, 1, 256, 4, 0),
    (3, [288], [64, 5, 30], [40, 300, 2], 2, 2, 192, 32, 0),
    (2, [128], [40, 64, 1, 1], [3, 200, 64, 0], 14, 2, 128, 128, 2),
    (3, [37, 51], [1, 2, 1, 4, 1, 1], [0, 1, 30, 2, 2, 200], 8, 2, 64, 16, 0),  # a prefix that ends within a page
]


@pytest.mark.parametrize("family,prefix,new,own,heads,kv,dim,page,alone", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("trees,by_head", [(False, False), (True, True)])
def test_matches_float64(family, prefix, new, own, heads, kv, dim, page, alone, dtype, trees, by_head):
    rng = np.random.default_rng([family, sum(prefix), sum(new), heads, dim])
    step = PrefixStep(rng, family, prefix, new, own, heads, kv, dim, page, dtype, alone, trees=trees, by_head=by_head)
    res = run(step, dtype)
    assert not res.status.any()


@pytest.mark.parametrize("family,n,heads,kv,dim", [(12, 1, 8, 1, 128), (4, 1, 4, 4, 64), (6, 9, 16, 2, 128),
                                                   (3, 2, 4, 2, 256), (16, 3, 4, 1, 192), (2, 1, 2, 1, 96)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_long_prefixes_are_split_and_joined(family, n, heads, kv, dim, dtype):
    rng = np.random.default_rng([family, n, heads, dim])
    own = list(rng.integers(0, 700, 2 * family + 1))
    run(PrefixStep(rng, family, [9000, 3000], [n] * (2 * family + 1), own, heads, kv, dim, 8, dtype, 1,
                   trees=n > 1), dtype)


@pytest.mark.parametrize("family,new,heads,kv,dim", [(2, 300, 4, 1, 64), (3, 130, 8, 2, 128), (2, 90, 2, 1, 256)])
def test_chunks(family, new, heads, kv, dim):
    rng = np.random.default_rng([family, new])
    run(PrefixStep(rng, family, [640], [new] * family, [int(x) for x in rng.integers(0, 200, family)], heads, kv, dim,
                   32, "bf16"), "bf16")


@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
def test_scales(scale):
    rng = np.random.default_rng(1)
    run(PrefixStep(rng, 4, [200], [2] * 4, [9, 0, 3, 70], 4, 2, 64, 8, "bf16"), "bf16", scale)


def test_the_same_as_tree_attention_on_requests_of_no_group():
    rng = np.random.default_rng(2)
    step = PrefixStep(rng, 1, [], [1, 5, 9], [100, 0, 40], 8, 2, 128, 16, "bf16", 3)
    a, vis = step.prefix_args()
    x, y = branches.prefix_attention(*a, lse=True), tree.tree_attention(*a[:6], lse=True)
    assert all(torch.equal(p, q) for p, q in zip(vars(x).values(), vars(y).values()))


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan"), 3e38])
@pytest.mark.parametrize("where", ["prefix", "own", "tree", "behind"])
def test_values_that_are_not_numbers(where, value):
    """In places that all, some or no rows see."""
    for family, new, dim in ((2, 3, 64), (6, 12, 128), (3, 20, 256)):
        rng = np.random.default_rng([new, dim])
        step = PrefixStep(rng, family, [200], [new] * family, [37] * family, 4, 2, dim, 8, "bf16", trees=True)
        ctx = int(step.kv_lengths[1]) - new
        at = dict(prefix=60, own=ctx - 5, tree=ctx + 1, behind=None)[where]
        if at is None:  # a page that no row holds, and what lies behind a request's last token
            rest = (ctx + new) % 8
            step.v[int(step.table[1, (ctx + new - 1) // 8]), rest or 7:, :, 3] = value if rest else 0
        else:
            step.v[int(step.table[1, at // 8]), at % 8, 0, 5] = value
        run(step, "bf16")


def test_masked_keys_that_are_not_numbers():
    rng = np.random.default_rng(3)
    step = PrefixStep(rng, 4, [104], [6] * 4, [20] * 4, 8, 2, 128, 8, "bf16")
    kv = int(step.kv_lengths[2])
    step.k[int(step.table[2, (kv - 1) // 8]), (kv - 1) % 8] = float("nan")  # seen by the last new token only
    args, _ = step.prefix_args()
    res = branches.prefix_attention(*args, lse=True)
    bad = torch.isnan(res.out).any(-1).any(-1)
    assert bad.nonzero()[:, 0].tolist() == [17]


def test_requests_that_are_refused():
    rng = np.random.default_rng(4)
    step = PrefixStep(rng, 3, [64, 96], [2] * 7, [30] * 7, 4, 2, 64, 16, "bf16", 1)
    step.kv_lengths[1] = 64 + 1   # its context is shorter than the prefix
    step.kv_lengths[4] = 1        # fewer than its new tokens
    args, _ = step.prefix_args()
    res = branches.prefix_attention(*args, lse=True)
    assert res.status.tolist() == [0, 16, 0, 0, 16, 0, 0]
    for r in (1, 4):
        assert not res.out[2 * r:2 * r + 2].any() and torch.isneginf(res.lse[2 * r:2 * r + 2]).all()
    many = PrefixStep(rng, 2, [32], [70, 3], [9, 9], 4, 2, 64, 16, "bf16")
    many.visible = np.full(73, 7, np.int64)  # more new tokens than a mask has bits
    more = branches.prefix_attention(*many.prefix_args()[0], visible=many.args()[1], lse=True)
    assert more.status.tolist() == [16, 0] and not more.out[:70].any() and torch.isneginf(more.lse[:70]).all()
    assert more.out[70:].any(-1).all()
    step.kv_lengths[[1, 4]] = step.kv_lengths[[0, 3]]
    fine = branches.prefix_attention(*step.prefix_args()[0], lse=True)
    keep = torch.tensor([0, 2, 3, 5, 6], device="cuda")
    rows = (keep[:, None] * 2 + torch.arange(2, device="cuda")).flatten()
    assert torch.equal(fine.out[rows], res.out[rows])


@pytest.mark.parametrize("groups,prefix,status", [
    ([0, 3, 6], [64, -1], [0, 0, 0, 16, 16, 16, 0]), ([0, 3, 6], [1 << 30, 96], [16, 16, 16, 0, 0, 0, 0]),
    ([0, 5, 3], [64, 64], [16] * 7), ([-1, 3, 6], [64, 64], [16] * 7), ([0, 3, 8], [64, 64], [16] * 7),
    ([1, 3, 3], [64, 64], [0] * 7), ([0, 0, 0], [64, 9], [0] * 7), ([7, 7, 7], [64, 9], [0] * 7),
    ([0, 7, 0, 7, 0, 7], [64] * 5, [16] * 7)])
def test_groups_out_of_bounds(groups, prefix, status):
    rng = np.random.default_rng(5)
    step = PrefixStep(rng, 3, [64, 96], [2] * 7, [30] * 7, 4, 2, 64, 16, "bf16", 1)
    whole = branches.prefix_attention(*step.prefix_args()[0], lse=True)
    step.groups, step.prefix = np.array(groups, np.int32), np.array(prefix, np.int32)
    res = branches.prefix_attention(*step.prefix_args()[0], lse=True)
    assert res.status.tolist() == status
    for r, s in enumerate(status):
        rows = slice(2 * r, 2 * r + 2)
        if s:
            assert not res.out[rows].any() and torch.isneginf(res.lse[rows]).all()
        else:  # the same row, joined from other parts
            # Two results, each off by 2^-8 of itself and of the values' mean size (below 4 together).
            assert (res.out[rows].float() - whole.out[rows].float()).abs().max() <= 2.0**-5
            assert (res.lse[rows] - whole.lse[rows]).abs().max() <= 1e-5


def test_pages_outside_the_cache_are_left_out():
    for new, dim in ((1, 64), (9, 128)):
        rng = np.random.default_rng([new, dim])
        step = PrefixStep(rng, 3, [96, 64], [new] * 7, [40] * 7, 4, 2, dim, 16, "bf16", 1)
        step.table[:3, 2] = -1                        # in the first group's prefix
        step.table[4, 6] = step.k.shape[0]            # behind the second's
        args, _ = step.prefix_args()
        res = branches.prefix_attention(*args, lse=True)
        assert res.status.tolist() == [20, 20, 20, 0, 20, 0, 0]
        check(step, res, "bf16")


def test_padding_rows_and_empty_requests():
    rng = np.random.default_rng(6)
    step = PrefixStep(rng, 2, [64], [0, 3, 0, 2], [9, 20, 5, 1], 4, 2, 64, 16, "f16", 2)
    args, _ = step.prefix_args()
    q = torch.cat([args[0].new_full((5, 4, 64), 7.0), args[0], args[0].new_full((9, 4, 64), 7.0)])
    out = torch.full_like(q, 3.0)
    res = branches.prefix_attention(q, *args[1:4], args[4] + 5, *args[5:], lse=True, out=out)
    assert not out[:5].any() and not out[10:].any()
    assert torch.isneginf(res.lse[:5]).all() and torch.isneginf(res.lse[10:]).all()
    # Tiles are chosen by the length of the arrays, so not bit by bit what a call without padding gives.
    check(step, tree.AttentionResult(out[5:10], res.lse[5:10], res.status), "f16")
    assert not res.status.any()
    # Fewer tokens than the offsets say: the last request has what there is of its own.
    for have in (1, 3, 4):
        cut = branches.prefix_attention(args[0][:have].contiguous(), *args[1:], lse=True)
        assert not cut.status.any() and torch.isfinite(cut.lse).all()
    none = branches.prefix_attention(q[:0], *args[1:4], torch.zeros_like(args[4]), *args[5:], lse=True)
    assert none.out.numel() == 0 and not none.status.any()


@pytest.mark.parametrize("n,dim", [(1, 64), (12, 128), (2, 256)])
def test_groups_with_empty_rows(n, dim):
    """Ended branches: rows without pages, tokens or a context, first ones of their group among them."""
    rng = np.random.default_rng([n, dim])
    new = [0, n, 0, n, 0, 0, 0, n, n]
    step = PrefixStep(rng, 4, [160, 96], new, [30] * 9, 4, 2, dim, 16, "bf16", 1)
    for r in (0, 4, 5, 6):
        step.table[r] = -1
        step.kv_lengths[r] = 0
    assert not run(step, "bf16").status.any()
    step.kv_lengths[[1, 7]] = 20 + n  # shorter than their prefixes: the next ones lead, or none
    args, _ = step.prefix_args()
    res = branches.prefix_attention(*args, lse=True)
    assert res.status.tolist() == [0, 16, 0, 0, 0, 0, 0, 16, 0]
    lo = step.offsets
    for r in (1, 7):
        assert not res.out[lo[r]:lo[r + 1]].any() and torch.isneginf(res.lse[lo[r]:lo[r + 1]]).all()
    want = tree.tree_attention(*args[:6], lse=True)
    for r in (3, 8):  # two results, each off by 2^-8 of itself and of the values' mean size (below 4 together)
        rows = slice(lo[r], lo[r + 1])
        assert (res.out[rows].float() - want.out[rows].float()).abs().max() <= 2.0**-5
        assert (res.lse[rows] - want.lse[rows]).abs().max() <= 1e-5


@pytest.mark.parametrize("family", [1, 7])
def test_many_requests(family):
    """More than every workgroup finds the groups of for itself."""
    rng = np.random.default_rng(family)
    R, alone = 1099, 1099 % family + 6 * family
    groups = (R - alone) // family
    prefix = [int(x) * 8 for x in rng.integers(0, 8, groups)]
    step = PrefixStep(rng, family, prefix, list(rng.integers(0, 3, R)), list(rng.integers(0, 20, R)), 2, 1, 64, 8,
                      "bf16", alone)
    assert not run(step, "bf16").status.any()
    step.groups[1::2], step.groups[::2] = R, 0  # all requests in every second group: nothing is read
    step.prefix[:] = 8
    res = branches.prefix_attention(*step.prefix_args()[0], lse=True)
    assert (res.status == 16).all() and not res.out.any() and torch.isneginf(res.lse).all()


@pytest.mark.parametrize("new", [1, 9])
def test_caches_past_32_bits(new):
    rng = np.random.default_rng(new)
    step = PrefixStep(rng, 4, [160, 96], [new] * 8, [30] * 8, 4, 2, 128, 16, "bf16")
    args, _ = step.prefix_args()
    near = branches.prefix_attention(*args, lse=True)
    far = branches.prefix_attention(args[0], far_apart(args[1]), far_apart(args[2]), *args[3:], lse=True)
    check(step, far, "bf16")
    assert torch.equal(far.out, near.out) and torch.equal(far.lse, near.lse) and not far.status.any()


def test_strided_rows_and_another_stream():
    rng = np.random.default_rng(7)
    step = PrefixStep(rng, 4, [320], [2] * 4, [50] * 4, 8, 2, 64, 16, "bf16")
    args, _ = step.prefix_args()
    packed = torch.zeros(8, 3, 8 * 64, device="cuda", dtype=torch.bfloat16)
    q = packed[:, 1].view(8, 8, 64)
    q.copy_(args[0])
    out = torch.zeros(8, 8, 2, 64, device="cuda", dtype=torch.bfloat16)[:, :, 1]
    want = branches.prefix_attention(*args, lse=True)
    p = branches.PreparedPrefixAttention(q, *args[1:], lse=True, out=out)
    p.launch()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.launch()
    torch.cuda.synchronize()
    assert torch.equal(out, want.out) and torch.equal(p.result.lse, want.lse)


def test_a_prepared_call_in_a_graph():
    rng = np.random.default_rng(8)
    step = PrefixStep(rng, 6, [800, 400], [3] * 12, list(rng.integers(0, 90, 12)), 8, 2, 128, 16, "bf16")
    args, _ = step.prefix_args()
    p = branches.PreparedPrefixAttention(*args, lse=True)
    p.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = p.launch()
    for turn in range(3):
        step.q = torch.randn_like(step.q)
        step.prefix = np.array([800 - 16 * turn, 400 - 32 * turn], np.int32)  # less of it is read once
        args[0].copy_(step.q)
        args[7].copy_(i32(step.prefix))
        got.out.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        check(step, got, "bf16")


def test_refusals():
    rng = np.random.default_rng(9)
    step = PrefixStep(rng, 2, [64], [1, 1], [9, 20], 4, 2, 64, 16, "bf16")
    args, _ = step.prefix_args()
    for i, bad in ((0, args[0].float()), (0, args[0][..., :60]), (1, args[1][:, :12]), (4, args[4][:2]),
                   (6, args[6].long()), (6, args[6][:0]), (6, i32([0, 1, 2, 2])), (7, args[7].repeat(2)),
                   (0, args[0].clone().requires_grad_())):
        with pytest.raises(ValueError):
            branches.prefix_attention(*args[:i], bad, *args[i + 1:])
    with pytest.raises(ValueError):
        branches.prefix_attention(*args, scale=float("nan"))
    with pytest.raises(TypeError):
        branches.prefix_attention(args[0].cpu(), *args[1:])
