"""Tensors that require a gradient: refused where it would be dropped, and the
inverse rotation as a training program uses it."""
import numpy as np
import pytest
import torch

from deepseekrpc_amd import tree
from oracle import tree_oracle as O
from tests.tree_util import Step, i32

pytestmark = pytest.mark.gpu


class Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, freqs, kw):
        ctx.saved = positions, freqs, kw
        return tree.rotary(x, None, positions, freqs, **kw).q

    @staticmethod
    def backward(ctx, grad):
        positions, freqs, kw = ctx.saved
        return tree.rotary(grad.contiguous(), None, positions, freqs, inverse=True, **kw).q, None, None, None


def test_rotary_does_not_drop_a_gradient():
    rng = np.random.default_rng(0)
    q, k, v = (torch.from_numpy(rng.standard_normal((5, 2, 16))).float().cuda() for _ in range(3))
    pos, (freqs, _) = i32(rng.integers(0, 1000, 5)), tree.rotary_frequencies(16)
    cache = dict(v=v, slots=i32(range(5)), k_cache=torch.zeros(2, 4, 2, 16, device="cuda"),
                 v_cache=torch.zeros(2, 4, 2, 16, device="cuda"))
    want = tree.rotary(q, k, pos, freqs)
    for t, call in ((q, lambda: tree.rotary(q, k, pos, freqs)), (k, lambda: tree.rotary(q, k, pos, freqs)),
                    (k, lambda: tree.PreparedRotary(None, k, pos, freqs)),
                    (v, lambda: tree.rotary(q, k, pos, freqs, **cache)),
                    (cache["k_cache"], lambda: tree.rotary(q, k, pos, freqs, **cache))):
        t.requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            call()
        t.requires_grad_(False)
        call()
    q.requires_grad_()
    assert torch.equal(tree.rotary(q.detach(), k, pos, freqs).q, want.q)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_in_a_training_program(interleaved):
    rng = np.random.default_rng(1)
    n, heads, dim, rot = 7, 3, 20, 12
    x = torch.from_numpy(rng.standard_normal((n, heads, dim))).float().cuda().requires_grad_()
    w = torch.from_numpy(rng.standard_normal((n, heads, dim))).float().cuda()
    pos, (freqs, _) = rng.integers(0, 5000, n), tree.rotary_frequencies(rot)
    y = Rotary.apply(x, i32(pos), freqs, dict(start=4, interleaved=interleaved, magnitude=1.2))
    (y * w).sum().backward()
    # The map is linear: its transpose applied to w, a basis vector at a time.
    eye = np.eye(heads * dim).reshape(-1, heads, dim)
    for t in range(n):
        jac = O.rotate(eye, [pos[t]] * (heads * dim), freqs.tolist(), 4, interleaved, False, 1.2)
        want = (jac * w[t].cpu().double().numpy()).sum((1, 2)).reshape(heads, dim)
        # Two products and a sum in float32 of terms up to 1.2 |w|, cosine and sine to 2^-23.
        assert np.abs(x.grad[t].cpu().double().numpy() - want).max() <= 8 * 2.0**-24 * 2.4 * float(w.abs().max())


def test_attention_does_not_drop_a_gradient():
    step = Step(np.random.default_rng(2), [2], [20], 4, 2, 64, 16, "bf16")
    args, _ = step.args()
    want = tree.tree_attention(*args).out
    for i in range(3):
        args[i].requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            tree.tree_attention(*args)
        with torch.no_grad():
            assert torch.equal(tree.tree_attention(*args).out, want)
        args[i].requires_grad_(False)
