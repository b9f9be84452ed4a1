"""The bound of tests/tree_exact.py itself, without a GPU: it stays near the
roundings that it stands for, and a coarser rounding of the weights passes it."""
import numpy as np
import pytest
import torch

from tests import tree_exact
from tests.tree_util import ROUND, Step

DIMS = (64, 128, 192, 256)


def rounded(dtype):
    return lambda p: torch.from_numpy(p).to(dtype).double().numpy()


@pytest.mark.parametrize("dim", DIMS)
def test_the_bound_is_a_few_roundings(dim):
    step = Step(np.random.default_rng(dim), [3], [400], 4, 2, dim, 16, "f16", trees=True, dev="cpu")
    out, _, bound, _ = tree_exact.attention(step, "f16")
    plain = tree_exact.attention(step, "f16", weights=rounded(torch.float16))[0]
    assert (np.abs(plain - out) <= bound).all()
    size = np.abs(step.v.double().numpy()).mean()  # about sum p |v|
    assert bound.max() < 4 * ROUND["f16"] * size
    step.q, step.k, step.v = (x.to(torch.bfloat16) for x in (step.q, step.k, step.v))
    assert tree_exact.attention(step, "bf16")[2].max() < 3 * ROUND["bf16"] * size


@pytest.mark.parametrize("dim", DIMS)
def test_weights_in_bf16_do_not_pass_for_f16(dim):
    step = Step(np.random.default_rng(dim), [4], [3], 8, 2, dim, 16, "f16", dev="cpu", spread=2.0)
    out, _, bound, _ = tree_exact.attention(step, "f16")
    wrong = tree_exact.attention(step, "f16", weights=rounded(torch.bfloat16))[0]
    assert (np.abs(wrong - out) > bound).any()
