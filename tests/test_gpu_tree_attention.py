"""dsr_tree_attention against float64 softmax attention, row by row, within
the bound of tests/tree_util.attention_bound."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import tree
from oracle import tree_oracle as O
from tests.tree_util import Step, attention_bound, i32

pytestmark = pytest.mark.gpu


def check(step, dtype, scale=None, call=None):
    args, vis = step.args()
    scale = step.dim ** -0.5 if scale is None else scale
    res = tree.tree_attention(*args, visible=vis, scale=scale, lse=True) if call is None else call
    q, k, v, *rest = step.host()
    out, lse, size = O.attention(q, k, v, *rest, scale)
    got, got_lse = res.out.float().cpu().numpy(), res.lse.cpu().numpy()
    kv = int(step.kv_lengths.max(initial=0))
    bound = attention_bound(dtype, out, size, q, k, scale, kv) if q.size else 0
    assert np.isfinite(got).all()
    assert (np.abs(got - out) <= bound).all(), float((np.abs(got - out) / bound).max())
    np.testing.assert_array_equal(np.isneginf(got_lse), np.isneginf(lse))
    fine = np.isfinite(lse)
    np.testing.assert_allclose(got_lse[fine], lse[fine], rtol=2e-6, atol=3e-5)
    return res


SHAPES = [  # new tokens, contexts, heads, kv heads, dim, page
    ([1], [0], 1, 1, 8, 1),
    ([1], [1], 4, 4, 64, 16),
    ([1], [31], 8, 2, 128, 16),
    ([1], [32], 8, 1, 128, 32),
    ([1], [700], 16, 1, 64, 64),
    ([1, 1, 1], [5, 0, 260], 10, 2, 96, 8),
    ([3, 0, 17], [33, 9, 1], 6, 3, 128, 4),
    ([16], [127], 4, 2, 72, 128),
    ([64, 5], [40, 300], 2, 1, 256, 16),
    ([33], [0], 7, 1, 192, 16),
    ([2, 63], [1025, 77], 32, 2, 128, 32),
    ([40, 64, 1], [3, 200, 64], 8, 1, 64, 16),
]


@pytest.mark.parametrize("new,ctx,heads,kv,dim,page", SHAPES)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("trees,by_head", [(False, False), (True, True)])
def test_matches_float64(new, ctx, heads, kv, dim, page, dtype, trees, by_head):
    rng = np.random.default_rng([sum(new), sum(ctx), heads, dim, page])
    res = check(Step(rng, new, ctx, heads, kv, dim, page, dtype, trees, by_head), dtype)
    assert not res.status.any()


@pytest.mark.parametrize("heads,kv,dim,n", [(8, 1, 128, 1), (16, 4, 64, 4), (8, 1, 128, 40), (4, 2, 256, 9),
                                             (4, 2, 192, 3), (6, 2, 96, 2), (4, 1, 192, 30)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_long_contexts_are_split_and_joined(heads, kv, dim, n, dtype):
    """Contexts that many workgroups share, next to ones that one takes alone."""
    rng = np.random.default_rng([heads, dim, n])
    ctx = [9000, 3, 2500, 0]
    check(Step(rng, [n, n, 1, n], ctx, heads, kv, dim, 16, dtype, trees=True), dtype)


@pytest.mark.parametrize("new,ctx", [([20, 18], [3000, 40]), ([31, 2, 25], [7, 0, 300])])
@pytest.mark.parametrize("dim,dtype", [(256, "bf16"), (248, "f16"), (192, "f16"), (136, "bf16")])
def test_wide_heads_of_some_rows(new, ctx, dim, dtype):
    """Between the smallest and the largest tiles, in parts and whole."""
    rng = np.random.default_rng([dim, ctx[0]])
    check(Step(rng, new, ctx, 4, 2, dim, 16, dtype, trees=True), dtype)
    check(Step(rng, new, ctx, 4, 2, dim, 1, dtype, by_head=True), dtype)


@pytest.mark.parametrize("new,ctx,heads,kv,dim,page", [
    ([300], [5000], 4, 1, 64, 16),             # a chunk behind a long context: in parts
    ([513, 0, 66], [0, 40, 0], 16, 2, 128, 32),  # whole tiles, the longest first
    ([700, 1], [0, 2000], 8, 1, 96, 1),
    ([130, 200], [100, 3], 3, 3, 256, 64),
])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_chunks_whole_and_in_parts(new, ctx, heads, kv, dim, page, dtype):
    rng = np.random.default_rng([sum(new), dim])
    res = check(Step(rng, new, ctx, heads, kv, dim, page, dtype), dtype)
    assert not res.status.any()


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
def test_one_long_request_has_many_parts(dim):
    rng = np.random.default_rng(dim)
    check(Step(rng, [1], [20_011], 4, 2, dim, 16, "bf16"), "bf16")


def test_many_requests():
    rng = np.random.default_rng(4)
    R = 200
    new, ctx = rng.integers(0, 4, R).tolist(), rng.integers(0, 90, R).tolist()
    new[0], ctx[7] = 0, 2000
    check(Step(rng, new, ctx, 4, 2, 64, 8, "bf16"), "bf16")


def test_long_chunks_of_a_prompt():
    """Without a mask more than 64 new tokens are a causal chunk."""
    rng = np.random.default_rng(6)
    check(Step(rng, [150, 1, 301], [0, 50, 33], 4, 2, 64, 16, "bf16"), "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_sharp_and_flat_rows(dtype):
    """Scores up to a few hundred (one token takes all, wherever it lies) and
    scores of zero (all tokens alike); a negative scale."""
    rng = np.random.default_rng(8)
    step = Step(rng, [4], [1500], 8, 2, 64, 16, dtype, spread=30.0)
    check(step, dtype)
    step.q.zero_()
    check(step, dtype)
    check(Step(rng, [4], [700], 8, 2, 64, 16, dtype), dtype, scale=-0.3)


def test_growing_maximum():
    """Keys whose scores rise along the context: the running maximum moves in
    every tile."""
    rng = np.random.default_rng(12)
    step = Step(rng, [1], [2000], 2, 1, 64, 16, "bf16")
    ramp = torch.linspace(-4, 4, 2001)
    flat = step.k.clone().zero_()
    at = np.arange(2001)
    flat[torch.from_numpy(step.table[0][at // 16].astype(np.int64)).cuda(), torch.from_numpy(at % 16).cuda(), 0] = \
        ramp[:, None].to(torch.bfloat16).cuda()
    step.k = flat
    step.q.fill_(3.0)
    check(step, "bf16")


@pytest.mark.parametrize("n", [20, 64])
def test_masks_that_leave_rows_empty(n):
    """No context and no visible node: zeros and -inf; a mask without the node
    itself; bits past the request's nodes are ignored."""
    rng = np.random.default_rng(n)
    step = Step(rng, [n, 5], [0, 40], 8, 2, 64, 16, "bf16", trees=True)
    words = step.visible.view(np.uint64).copy()
    words[0] = 0
    words[3] = 0
    words[4] = 1 << 2
    words[n] = 0
    words[n + 1] = 0xFFFFFFFFFFFFFFE0
    step.visible = words.view(np.int64)
    keep = step.visible.copy()
    step.visible = np.where(np.arange(n + 5) == n + 1, 0, step.visible)  # what the extra bits must mean
    want = step.host()
    step.visible = keep
    args, vis = step.args()
    res = tree.tree_attention(*args, visible=vis, lse=True)
    out, lse, size = O.attention(*want, 64 ** -0.5)
    got = res.out.float().cpu().numpy()
    assert (got[[0, 3]] == 0).all() and torch.isneginf(res.lse[[0, 3]]).all()
    assert (np.abs(got - out) <= attention_bound("bf16", out, size, want[0], want[1], 64 ** -0.5, 50)).all()


@pytest.mark.parametrize("what", [float("inf"), float("nan"), -float("inf")])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("new", [[6], [40]])
def test_what_masked_places_hold_never_reaches_a_row(what, dtype, new):
    """Infinities and NaN in keys and values of nodes a row does not see, in
    the page behind the last token and in pages of no request."""
    rng = np.random.default_rng(21)
    step = Step(rng, new, [70], 4, 2, 64, 16, dtype, trees=True)
    n, page = new[0], 16
    clean = check(step, dtype)
    word = step.visible.view(np.uint64)
    poisoned = 3  # this node's row is bad: only rows that see it may show it
    slot = lambda p: (int(step.table[0, p // page]), p % page)  # noqa: E731
    for c in (step.k, step.v):
        used = np.zeros((c.shape[0], page), bool)
        for p in range(70 + n):
            used[slot(p)] = True
        c[torch.from_numpy(~used).cuda()] = what
    b, o = slot(70 + poisoned)
    step.v[b, o, :, ::3] = what
    step.k[b, o, 0] = what
    args, vis = step.args()
    res = tree.tree_attention(*args, visible=vis, lse=True)
    unseen = torch.from_numpy(np.array([not int(w) >> poisoned & 1 for w in word])).cuda()
    assert unseen.any() and (~unseen).any()
    assert torch.equal(res.out[unseen], clean.out[unseen]) or \
        torch.allclose(res.out[unseen].float(), clean.out[unseen].float(), rtol=2**-7, atol=1e-3)
    assert torch.isfinite(res.out[unseen]).all()
    assert torch.equal(res.lse[unseen], clean.lse[unseen])
    assert not torch.isfinite(res.out[~unseen][..., ::3]).all()


def test_bad_lengths_and_pages():
    """Statuses; the other requests are served."""
    rng = np.random.default_rng(30)
    step = Step(rng, [3, 3, 3, 3, 1], [100, 50, 2000, 60, 10], 4, 2, 64, 16, "bf16")
    args, _ = step.args()
    good = tree.tree_attention(*args, lse=True)
    table, kv = args[3].clone(), args[5].clone()
    kv[0] = 2                          # fewer cached tokens than new ones
    kv[1] = table.shape[1] * 16 + 1    # more than a table row
    table[2, 7] = step.k.shape[0]
    table[3, 1] = -5
    res = tree.tree_attention(*args[:3], table, args[4], kv, lse=True)
    assert res.status.tolist() == [O.E_LENGTH, O.E_LENGTH, O.E_BLOCK, O.E_BLOCK, 0]
    assert not res.out[:6].any() and torch.isneginf(res.lse[:6]).all()
    assert torch.equal(res.out[12:], good.out[12:])
    # The pages outside the cache are left out.
    host = step.host()
    for r, page in ((2, 7), (3, 1)):
        rows = slice(3 * r, 3 * r + 3)
        total = int(step.kv_lengths[r])
        seen = [p for p in range(total) if p // 16 != page]
        one = np.zeros((1, len(seen)), np.int32)
        q, k, v = host[0][rows], host[1], host[2]
        kk = k[step.table[r, np.array(seen) // 16], np.array(seen) % 16][:, None]
        vv = v[step.table[r, np.array(seen) // 16], np.array(seen) % 16][:, None]
        one[0] = np.arange(len(seen))
        out, lse, size = O.attention(q, kk, vv, one, [0, 3], [len(seen)], None, 0.125)
        bound = attention_bound("bf16", out, size, q, k, 0.125, total)
        assert (np.abs(res.out[rows].float().cpu().numpy() - out) <= bound).all()
    many = Step(rng, [65], [3], 2, 1, 64, 16, "bf16")
    a, _ = many.args()
    res = tree.tree_attention(*a, visible=torch.ones(65, dtype=torch.int64, device="cuda"))
    assert res.status.tolist() == [O.E_LENGTH] and not res.out.any()


@pytest.mark.parametrize("new,ctx", [(150, 0), (200, 1500)])
def test_bad_page_that_only_a_chunks_last_rows_see(new, ctx):
    """Causal rows are tiled, and the first tiles end before the last page."""
    step = Step(np.random.default_rng(new), [new, 7], [ctx, 90], 8, 2, 64, 16, "bf16")
    step.table[0, (ctx + new - 1) // 16] = step.k.shape[0]
    args, vis = step.args()
    res = tree.tree_attention(*args, visible=vis, scale=0.125)
    assert res.status.tolist() == [O.E_BLOCK, 0]


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements whose used pages lie at its end."""
    rng = np.random.default_rng(31)
    blocks, page, kv, dim = 70_000, 32, 8, 128  # 2.3e9 elements
    step = Step(rng, [2], [300], 16, kv, dim, page, "bf16")
    small = step.k.shape[0]
    big = [torch.empty(blocks, page, kv, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for b, c in zip(big, (step.k, step.v)):
        b[blocks - small:] = c
    args, _ = step.args()
    table = torch.where(args[3] >= 0, args[3] + blocks - small, args[3])
    a = tree.tree_attention(*args, lse=True)
    b = tree.tree_attention(args[0], *big, table, *args[4:], lse=True)
    assert torch.equal(a.out, b.out) and torch.equal(a.lse, b.lse)


def test_strides_out_tensor_and_repeats():
    """Packed queries, an output tensor with strides, repeated launches: the
    same bits each time."""
    rng = np.random.default_rng(33)
    step = Step(rng, [5, 9], [800, 40], 8, 2, 64, 16, "bf16", trees=True)
    args, vis = step.args()
    want = tree.tree_attention(*args, visible=vis, lse=True)
    wide = torch.randn(14, 12, 72, device="cuda").to(torch.bfloat16)
    wide[:, 2:10, 8:] = args[0]
    out = torch.zeros(14, 9, 128, device="cuda", dtype=torch.bfloat16)
    call = tree.PreparedTreeAttention(wide[:, 2:10, 8:], *args[1:], visible=vis, lse=True, out=out[:, 1:, 32:96])
    for _ in range(3):
        res = call.launch()
        assert torch.equal(res.out, want.out) and torch.equal(res.lse, want.lse)
    assert not out[:, 0].any() and not out[..., :32].any() and not out[..., 96:].any()


def test_another_stream_and_a_graph():
    rng = np.random.default_rng(34)
    step = Step(rng, [4] * 6, [3000, 10, 500, 0, 77, 1234], 8, 2, 128, 16, "bf16", trees=True)
    args, vis = step.args()
    call = tree.PreparedTreeAttention(*args, visible=vis, lse=True)
    want = [t.clone() for t in vars(call.launch()).values()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call.launch()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(vars(call.result).values(), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        call.launch()  # binds this stream's scratch before the capture
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        call.launch()
    for turn in range(4):
        call.result.out.zero_()
        args[0].mul_(-1)  # other queries: replays read what the tensors hold now
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in vars(call.result).values()]
        call.launch()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, vars(call.result).values())), turn


def test_no_tokens_and_refused_arguments():
    rng = np.random.default_rng(35)
    step = Step(rng, [2], [20], 4, 2, 64, 16, "bf16")
    args, _ = step.args()
    q, k, v, table, off, kv = args
    none = tree.tree_attention(q[:0], k, v, table, i32([0, 0]), kv, lse=True)
    assert none.out.shape == (0, 4, 64) and none.status.tolist() == [0]
    vis = torch.ones(2, dtype=torch.int64, device="cuda")
    f32 = [t.float() for t in (q, k, v)]
    for a, kw in ((f32 + [table, off, kv], {}), ((q, k.half(), v, table, off, kv), {}),
                  ((q, k, v[:1], table, off, kv), {}), ((q[:, :3], k, v, table, off, kv), {}),
                  ((q[..., :60], k[..., :60], v[..., :60], table, off, kv), {}),
                  ((q, k, v, table.long(), off, kv), {}), ((q, k, v, table, off[:1], kv), {}),
                  ((q, k, v, table, off.long(), kv), {}), ((q, k, v, table, off, kv.cpu()), {}),
                  ((q, k[:, :12], v[:, :12], table, off, kv), {}), ((q, k, v, table[:0], off, kv), {}),
                  ((q, k, v, table, off, kv), dict(visible=vis.int())),
                  ((q, k, v, table, off, kv), dict(visible=vis[:1])),
                  ((q, k, v, table, off, kv), dict(scale=float("inf"))),
                  ((q, k, v, table, off, kv), dict(out=q.float())),
                  ((q.cpu(), k, v, table, off, kv), {})):
        with pytest.raises((TypeError, ValueError)):
            tree.tree_attention(*a, **kw)
    odd = torch.empty(2 * 4 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(2, 4, 64)
    with pytest.raises(ValueError):
        tree.tree_attention(odd, k, v, table, off, kv)


# The calls above are small, and few-row tiles take them.  Many tiles, or table
# rows with room for long contexts, bring the kernels with larger tiles.


@pytest.mark.parametrize("dim,heads,kv,most", [(128, 64, 8, 5), (72, 64, 8, 5), (64, 32, 8, 20), (128, 32, 8, 20),
                                               (96, 24, 8, 20), (192, 64, 8, 5), (256, 32, 8, 9), (136, 16, 8, 9),
                                               (256, 64, 8, 20)])
@pytest.mark.parametrize("longest,page,trees,by_head", [(100, 32, True, False), (2100, 16, False, True),
                                                        (2300, 1, True, False)])
def test_many_tiles(dim, heads, kv, most, longest, page, trees, by_head):
    """Whole (short table rows) and in parts, each with one long request among short ones."""
    rng = np.random.default_rng([dim, heads, most, longest])
    R = 72
    new, ctx = rng.integers(1, most + 1, R).tolist(), rng.integers(0, 40, R).tolist()
    ctx[11], new[30] = longest, 0
    check(Step(rng, new, ctx, heads, kv, dim, page, "f16" if dim in (72, 192) else "bf16", trees, by_head),
          "f16" if dim in (72, 192) else "bf16")


def roomy(step):
    """The step's arguments with table rows of about four million tokens."""
    args, vis = Step.plain_args(step)
    columns = (1 << 22) // step.page - args[3].shape[1]
    table = torch.nn.functional.pad(args[3], (0, columns), value=-1)
    return (*args[:3], table, *args[4:]), vis


AGAIN = ([(test_matches_float64, (*shape, dtype, *how)) for shape in SHAPES for dtype in ("bf16", "f16")
          for how in ((False, False), (True, True))]
         + [(test_long_contexts_are_split_and_joined, (h, k, d, n, "bf16"))
            for h, k, d, n in ((8, 1, 128, 3), (8, 1, 128, 40), (8, 1, 64, 4), (4, 1, 192, 9), (4, 2, 256, 30))]
         + [(test_sharp_and_flat_rows, (dtype,)) for dtype in ("bf16", "f16")]
         + [(test_growing_maximum, ()), (test_bad_lengths_and_pages, ()), (test_long_chunks_of_a_prompt, ())]
         + [(test_masks_that_leave_rows_empty, (n,)) for n in (20, 64)]
         + [(test_what_masked_places_hold_never_reaches_a_row, (what, dtype, new))
            for what in (float("inf"), float("nan")) for dtype in ("bf16", "f16") for new in ([12], [40])]
         + [(test_wide_heads_of_some_rows, ([20, 18], [300, 40], dim, "f16")) for dim in (192, 256)]
         + [(test_bad_page_that_only_a_chunks_last_rows_see, (150, 0))])


@pytest.mark.parametrize("case", range(len(AGAIN)))
def test_again_with_larger_tiles(case, monkeypatch):
    test, args = AGAIN[case]
    monkeypatch.setattr(Step, "plain_args", Step.args, raising=False)
    monkeypatch.setattr(Step, "args", roomy)
    test(*args)
