"""dsr_rotary against float64 rotations.

Bounds: a rotated value carries one rounding to its type and a few float32
ones (cosine, sine, two products, one sum: at most 4 x 2^-24 of |a| + |b|,
and the angle's 2^-24 half turns), so |error| <= u |y| + 8 x 2^-24 (|a| + |b|)
magnitude."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import tree
from oracle import tree_oracle as O
from tests.tree_util import DTYPES, ROUND, i32

pytestmark = pytest.mark.gpu


def f64(t):
    return t.detach().cpu().double().numpy()


def close(got, want, x, dtype, magnitude=1.0):
    bound = ROUND[dtype] * np.abs(want) + 8 * 2.0**-24 * 2 * np.abs(x).max() * magnitude + 1e-12
    err = np.abs(got - want)
    assert (err <= bound).all(), float((err / bound).max())


def normal(rng, dtype, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).cuda().to(DTYPES[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot,start", [(1, 1, 1, 2, 2, 0), (1, 8, 2, 64, 64, 0),
                                                           (3, 4, 1, 128, 64, 64), (70, 5, 5, 80, 40, 40),
                                                           (33, 3, 3, 24, 6, 3), (9, 2, 1, 512, 512, 0),
                                                           (1200, 6, 2, 96, 48, 0)])
def test_forward_and_inverse(dtype, interleaved, tokens, heads, kv, dim, rot, start):
    rng = np.random.default_rng([tokens, dim, rot, start, interleaved])
    q, k = normal(rng, dtype, tokens, heads, dim), normal(rng, dtype, tokens, kv, dim)
    pos = rng.integers(0, 3_000_000, tokens)
    pos[0] = 0
    freqs, _ = tree.rotary_frequencies(rot)
    for inverse in (False, True):
        res = tree.rotary(q, k, i32(pos), freqs, start=start, interleaved=interleaved, inverse=inverse, magnitude=1.25)
        for got, x in ((res.q, q), (res.k, k)):
            want = O.rotate(f64(x), pos, freqs.tolist(), start, interleaved, inverse, 1.25)
            close(f64(got), want, f64(x), dtype, 1.25)
            keep = [d for d in range(dim) if not start <= d < start + rot]
            assert torch.equal(got[..., keep], x[..., keep])


@pytest.mark.parametrize("dtype,by_head,page,v_dim", [("bf16", False, 16, 64), ("f16", True, 1, 40), ("f32", False, 8, 64),
                                                      ("bf16", True, 128, 3)])
def test_cache_writes(dtype, by_head, page, v_dim):
    """Rotated keys and values land in their slots and nowhere else; padding
    tokens write nothing; slots outside the cache give a status."""
    rng = np.random.default_rng([page, v_dim])
    n, heads, kv, dim, rot = 37, 6, 3, 64, 32
    blocks = 200 // page + 2
    packed = normal(rng, dtype, n, (heads + kv) * dim + kv * v_dim)
    q = packed[:, :heads * dim].view(n, heads, dim)
    k = packed[:, heads * dim:(heads + kv) * dim].view(n, kv, dim)
    v = packed[:, (heads + kv) * dim:].view(n, kv, v_dim)
    shape = lambda d: (blocks, kv, page, d) if by_head else (blocks, page, kv, d)  # noqa: E731
    kc, vc = normal(rng, dtype, *shape(dim)), normal(rng, dtype, *shape(v_dim))
    kc, vc = (t.transpose(1, 2) if by_head else t for t in (kc, vc))
    old_k, old_v = kc.clone(), vc.clone()
    slots = rng.permutation(blocks * page)[:n]
    slots[4], slots[9], slots[11], slots[20] = -1, blocks * page, -7, 2**31 - 1
    pos = rng.integers(0, 100_000, n)
    freqs, _ = tree.rotary_frequencies(rot)
    res = tree.rotary(q, k, i32(pos), freqs, v=v, start=8, slots=i32(slots), k_cache=kc, v_cache=vc)
    want_status = np.zeros(n, int)
    want_status[[9, 11, 20]] = O.E_BLOCK
    np.testing.assert_array_equal(res.status.cpu().numpy(), want_status)
    assert res.k is None
    close(f64(res.q), O.rotate(f64(q), pos, freqs.tolist(), 8, False, False, 1.0), f64(q), dtype)
    rk = O.rotate(f64(k), pos, freqs.tolist(), 8, False, False, 1.0)
    touched = torch.zeros(blocks, page, dtype=torch.bool)
    for i, s in enumerate(slots):
        if 0 <= s < blocks * page:
            close(f64(kc[s // page, s % page]), rk[i], f64(k), dtype)
            assert torch.equal(vc[s // page, s % page], v[i])
            touched[s // page, s % page] = True
    assert torch.equal(kc[~touched], old_k[~touched]) and torch.equal(vc[~touched], old_v[~touched])


def test_in_place_and_queries_or_keys_alone():
    rng = np.random.default_rng(3)
    for dtype, dim, start in (("bf16", 64, 0), ("f32", 30, 5)):
        x = normal(rng, dtype, 50, 4, dim)
        pos, (freqs, _) = i32(rng.integers(0, 5000, 50)), tree.rotary_frequencies(20 if dim == 30 else 32)
        want = tree.rotary(x, None, pos, freqs, start=start).q
        only_k = tree.rotary(None, x, pos, freqs, start=start)
        assert only_k.q is None and torch.equal(only_k.k, want)
        y, z = x.clone(), x.clone()
        res = tree.rotary(y, z, pos, freqs, start=start, q_out=y, k_out=z)
        assert res.q is y and torch.equal(y, want) and torch.equal(z, want)
        wide = torch.zeros(50, 4, 2 * dim, dtype=x.dtype, device="cuda")
        tree.rotary(x, None, pos, freqs, start=start, q_out=wide[..., dim:] if dim == 64 else wide[..., 1:dim + 1])
        assert torch.equal(wide[..., dim:] if dim == 64 else wide[..., 1:dim + 1], want)


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_gradient(interleaved):
    """d sum(w . rotary(x)) / dx is the inverse rotation of w: against the
    float64 formula's transpose, and against central differences of the
    forward kernel (linear in x, so a difference over 2 h is the derivative up
    to float32 rounding: 2^-22 |y| / h per term)."""
    rng = np.random.default_rng(17)
    n, heads, dim, rot, start, m = 5, 2, 12, 8, 2, 1.5
    x, w = normal(rng, "f32", n, heads, dim), normal(rng, "f32", n, heads, dim)
    pos = rng.integers(0, 40_000, n)
    freqs, _ = tree.rotary_frequencies(rot)
    kw = dict(start=start, interleaved=interleaved, magnitude=m)
    grad = f64(tree.rotary(w, None, i32(pos), freqs, inverse=True, **kw).q)
    eye = np.eye(heads * dim).reshape(heads * dim, heads, dim)
    for t in range(n):
        jac = O.rotate(eye, [pos[t]] * (heads * dim), freqs.tolist(), start, interleaved, False, m)
        want = (jac * f64(w)[t]).sum((1, 2)).reshape(heads, dim)
        assert np.abs(grad[t] - want).max() < 1e-5
    h = 0.25
    for h_i in range(heads):
        for d in range(dim):
            e = torch.zeros_like(x)
            e[:, h_i, d] = h
            up, down = (f64(tree.rotary(x + s * e, None, i32(pos), freqs, **kw).q) for s in (1, -1))
            slope = ((up - down) * f64(w)).sum((1, 2)) / (2 * h)
            assert np.abs(slope - grad[:, h_i, d]).max() < 1e-4


def test_frequencies():
    f, m = tree.rotary_frequencies(8, 10000.0, device="cpu")
    np.testing.assert_allclose(f, 10000.0 ** (-np.arange(4) / 4), rtol=1e-12)
    assert m == 1.0 and f.dtype == torch.float64
    g, _ = tree.rotary_frequencies(8, scaling="linear", factor=4.0, device="cpu")
    np.testing.assert_allclose(g, f / 4)
    g, _ = tree.rotary_frequencies(8, scaling="base", factor=4.0, device="cpu")
    np.testing.assert_allclose([g[0], g[-1]], [f[0], f[-1] / 4])
    g, m = tree.rotary_frequencies(64, scaling="ramp", factor=8.0, original=4096, device="cpu")
    f, _ = tree.rotary_frequencies(64, device="cpu")
    turns = 4096 * f / (2 * np.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.allclose(g[turns <= 1], f[turns <= 1] / 8)
    assert ((g <= f) & (g >= f / 8)).all() and abs(m - 1 - 0.1 * np.log(8)) < 1e-12
    for bad in (dict(rot_dim=7), dict(rot_dim=8, base=1.0), dict(rot_dim=8, factor=0.5), dict(rot_dim=8, scaling="x")):
        with pytest.raises(ValueError):
            tree.rotary_frequencies(device="cpu", **bad)


def test_refused_arguments():
    rng = np.random.default_rng(1)
    q, k, v = (normal(rng, "bf16", 4, h, 16) for h in (4, 2, 2))
    pos, (freqs, _) = i32([0, 1, 2, 3]), tree.rotary_frequencies(16)
    kc, vc = normal(rng, "bf16", 3, 8, 2, 16), normal(rng, "bf16", 3, 8, 2, 16)
    slots = i32([0, 1, 2, 3])
    tree.rotary(q, k, pos, freqs, v=v, slots=slots, k_cache=kc, v_cache=vc)
    full = dict(v=v, slots=slots, k_cache=kc, v_cache=vc)
    for a, kw in (((q.cpu(), k, pos, freqs), {}), ((q.double(), k, pos, freqs), {}), ((q, k.float(), pos, freqs), {}),
                  ((q, k[:3], pos, freqs), {}), ((q, k, pos.long(), freqs), {}), ((q, k, pos, freqs.float()), {}),
                  ((q, k, pos, freqs), dict(start=2)), ((q, k, pos, freqs), dict(start=-1)),
                  ((q, k, pos, freqs), dict(magnitude=0.0)), ((q, k, pos, freqs), dict(magnitude=float("nan"))),
                  ((q, k, pos, freqs), dict(full, slots=None)), ((q, k, pos, freqs), dict(full, v=None)),
                  ((q, None, pos, freqs), full), ((q, k, pos, freqs), dict(full, v_cache=vc[:2])),
                  ((q, k, pos, freqs), dict(full, k_cache=kc[:, :6])), ((q, k, pos, freqs), dict(k_out=q)),
                  ((q, k, pos, freqs), dict(q_out=q.transpose(0, 1))), ((None, k, pos, freqs), dict(q_out=q)),
                  ((q.transpose(1, 2), None, pos, freqs), {})):
        with pytest.raises((TypeError, ValueError)):
            tree.rotary(*a, **kw)
    empty = tree.rotary(q[:0], k[:0], pos[:0], freqs)
    assert empty.q.shape == (0, 4, 16)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot,start", [(11, 4, 2, 64, 24, 0), (1100, 3, 3, 20, 8, 4),
                                                           (5, 2, 1, 128, 40, 84)])
def test_rows_that_only_8_byte_accesses_fit(dtype, interleaved, tokens, heads, kv, dim, rot, start):
    test_forward_and_inverse(dtype, interleaved, tokens, heads, kv, dim, rot, start)


@pytest.mark.parametrize("dtype,by_head,page,v_dim", [("bf16", False, 16, 20), ("f16", True, 1, 12)])
def test_cache_writes_of_8_byte_rows(dtype, by_head, page, v_dim):
    test_cache_writes(dtype, by_head, page, v_dim)
