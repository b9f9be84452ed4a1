"""The speculative loop of examples/tree_decode.py: greedy ids are those of
decoding one token at a time, in fewer steps, and every page comes back."""
import numpy as np
import pytest
import torch

from examples import tree_decode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [1, 16])
def test_greedy_trees_decode_as_single_tokens_do(page):
    model = tree_decode.Model()
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, 512, n).tolist() for n in (3, 1, 70, 18, 33)]
    one = tree_decode.generate(model, prompts, 40, drafts=False, page=page)
    many = tree_decode.generate(model, prompts, 40, page=page)
    assert [o.ids for o in one] == [o.ids for o in many] and all(len(o.ids) == 40 for o in many)
    assert sum(o.steps for o in many) < 0.8 * sum(o.steps for o in one)


def test_sampled_trees_stay_in_bounds():
    model = tree_decode.Model(seed=1)

    def uniforms(step, rows):
        return torch.from_numpy(np.random.default_rng([step, rows]).random(rows)).cuda()

    out = tree_decode.generate(model, [[1, 2, 3], [9]], 30, policy=dict(temperature=0.8, top_k=20), uniforms=uniforms)
    assert all(len(o.ids) == 30 and all(0 <= t < 512 for t in o.ids) for o in out)
