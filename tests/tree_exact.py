"""Attention of the tree tests in float64, row by row, with an error bound from
each row's own scores."""
import numpy as np

from tests.tree_util import ROUND


def sees(step, r, t):
    """Which of request r's cached tokens its new token t sees."""
    lo, hi, kv = int(step.offsets[r]), int(step.offsets[r + 1]), int(step.kv_lengths[r])
    at, ctx = np.arange(kv), kv - (hi - lo)
    if step.visible is None:
        see = at <= ctx + t
    else:
        word = int(np.int64(step.visible[lo + t]).view(np.uint64))
        see = np.array([j < ctx or bool(word >> int(j - ctx) & 1) for j in at], bool)
    page = step.table[r, at // step.page]
    return see & (page >= 0) & (page < step.k.shape[0])  # what lies outside the cache is left out


def attention(step, dtype, scale=None, weights=lambda p: p):
    """out, lse, and the bounds of both.  ``weights`` plants a mistake.

    With u the rounding of the rows' type and e = 2^-24 of float32, a score
    s = scale sum q_d k_d carries dim e scale sum |q_d k_d| from its sum, a few e
    |s| from the scale's two roundings and the base's subtraction, and its
    exponential and the factors that parts are joined with a few e more (at
    most 20: one for each time the maximum passes the last by 2^8, each wave
    and each part).  The sums are of at most kv / 8 + 64 terms in a row.  The
    weights are rounded to the type for the values only, and the output is."""
    q, k, v = (x.cpu().double().numpy() for x in (step.q, step.k, step.v))
    n, heads, dim = q.shape
    group = heads // k.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    u, e = ROUND[dtype], 2.0**-24
    out, bound = np.zeros((2, n, heads, dim))
    lse, lse_bound = np.full((n, heads), -np.inf), np.zeros((n, heads))
    for r in range(len(step.kv_lengths)):
        lo, hi = int(step.offsets[r]), int(step.offsets[r + 1])
        for t in range(hi - lo):
            at = np.flatnonzero(sees(step, r, t))
            if not len(at):
                continue
            kk, vv = (x[step.table[r, at // step.page], at % step.page] for x in (k, v))
            for h in range(heads):
                s = kk[:, h // group] @ q[lo + t, h] * scale
                top = s.max()
                p = np.exp(s - top)
                total = p.sum()
                p /= total
                far = dim * e * (np.abs(kk[:, h // group]) @ np.abs(q[lo + t, h])) * abs(scale)
                far += e * (8 * np.abs(s) + 4 * (top - s) + 40)
                chain = e * (len(at) / 8 + 64)
                w = vv[:, h // group]
                with np.errstate(invalid="ignore"):
                    o = (weights(p)[:, None] * w).sum(0)
                    size = ((p * (u + far + chain))[:, None] * np.abs(w)).sum(0)
                    out[lo + t, h] = o
                    bound[lo + t, h] = 1.02 * (size + np.abs(o) * (u + p @ far + chain)) + 2.0**-25 * (dtype == "f16")
                lse[lo + t, h] = top + np.log(total)
                lse_bound[lo + t, h] = 1.02 * (p @ far + chain) + 8 * e * abs(lse[lo + t, h]) + 8 * e
    return out, lse, bound, lse_bound


def check(step, res, dtype, scale=None):
    """The kernel's results: infinities and NaN where they belong, the rest
    within the bound."""
    out, lse, bound, lse_bound = attention(step, dtype, scale)
    got, got_lse = res.out.cpu().double().numpy(), res.lse.cpu().double().numpy()
    for kind in (np.isnan, np.isposinf, np.isneginf):
        np.testing.assert_array_equal(kind(got), kind(out), err_msg=kind.__name__)
    fine = np.isfinite(out)
    ratio = np.abs(got[fine] - out[fine]) / np.maximum(bound[fine], 1e-300)
    assert (ratio <= 1).all(), float(ratio.max())
    np.testing.assert_array_equal(np.isneginf(got_lse), np.isneginf(lse))
    seen = np.isfinite(lse)
    assert (np.abs(got_lse[seen] - lse[seen]) <= lse_bound[seen]).all()
    return out
