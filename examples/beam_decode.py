"""Beam search over a paged cache: the operators of branches in one loop.

The small random transformer of tree_decode continues each prompt with several
beams.  A prompt is ingested once; then its beams are rows that share its pages,
and every step

  select_beams -> fork_pages -> plan_blocks
  -> per layer (rotary with cache writes -> prefix_attention) -> vocab_head

continues them.  Tables, page pool, scores and the beams' tokens stay on the
device.

    python examples/beam_decode.py
"""
import functools
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from deepseekrpc_amd import branches, tree  # noqa: E402
from examples.tree_decode import Model  # noqa: E402


def search(model, prompts, new_tokens, beams, *, page=16, eos=None, compact_every=0):
    """For each prompt its ``beams`` best continuations of up to ``new_tokens``
    ids: ``(ids, score)`` lists, best first, and the pages free at the end and
    in all."""
    dev, R, rows = model.device, len(prompts), len(prompts) * beams
    width = -(-(max(map(len, prompts)) + new_tokens) // page)
    blocks = R * width + rows * (new_tokens // page + 2)
    shape = (blocks, page, model.kv, model.head)
    k_caches = [torch.zeros(shape, dtype=torch.bfloat16, device=dev) for _ in range(model.layers)]
    v_caches = [torch.zeros_like(t) for t in k_caches]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    pool, state = tree.page_pool(blocks, dev)
    shared = torch.zeros(blocks, dtype=torch.int32, device=dev)
    table = torch.full((R, width), -1, dtype=torch.int32, device=dev)

    # Prompts, a row each: one causal chunk.
    flat = i32([t for p in prompts for t in p])
    plan = tree.plan_blocks(i32([0] * R), i32([len(p) for p in prompts]), table, i32([0] * R), pool, state,
                            blocks=blocks, page=page, capacity=flat.numel())
    hidden = model.forward(flat, plan, k_caches, v_caches)
    logits = model.logits(hidden[plan.offsets[1:].long() - 1])
    held, lengths = plan.held, plan.kv_lengths
    scores = torch.zeros(R, dtype=torch.float64, device=dev)
    offsets = torch.arange(R + 1, dtype=torch.int32, device=dev)
    finished = torch.zeros(R, dtype=torch.int32, device=dev)
    ids = torch.zeros(R, 0, dtype=torch.int32, device=dev)

    # The whole pages of a prompt are what its beams have in common.
    groups = offsets * beams
    attend = functools.partial(branches.prefix_attention, groups=groups,
                               prefix_lengths=i32([len(p) // page * page for p in prompts]))
    for step in range(new_tokens):
        best = branches.select_beams(logits, scores, offsets, keep=beams, finished=finished)
        parents, tokens = best.parents.flatten(), best.tokens.flatten()
        fork = branches.fork_pages(lengths, parents, table, held, shared, pool, state, [*k_caches, *v_caches])
        table, held, lengths = fork.table, fork.held, fork.lengths
        if compact_every and step % compact_every == 0:
            branches.compact_pages(table, held, pool, state, [*k_caches, *v_caches], shared=shared)
        source = parents.long().clamp(min=0)
        ended = (tokens < 0) | (finished[source] != 0)
        ids = torch.cat([ids[source], tokens[:, None]], 1)
        finished = ended | (tokens == eos) if eos is not None else ended
        finished = finished.to(torch.int32)
        scores, offsets = best.scores.flatten(), groups
        # A token each of the rows that go on; capacity is for all of them.
        plan = tree.plan_blocks(lengths, 1 - finished, table, held, pool, state, blocks=blocks, page=page,
                                capacity=rows)
        owner = plan.owners.long()
        hidden = model.forward(torch.where(owner < 0, 0, tokens[owner]), plan, k_caches, v_caches, attend)
        # Logits of each row that brought a token, where the row is.
        at = plan.offsets[:-1].long().clamp(max=rows - 1)
        logits = model.logits(hidden[at])
        lengths = plan.kv_lengths
    out, ids, scores = [], ids.tolist(), scores.tolist()
    for r in range(R):
        out.append([([t for t in ids[i] if t >= 0], scores[i]) for i in range(r * beams, (r + 1) * beams)
                    if scores[i] > float("-inf")])
    # No row goes on: every page comes back.
    branches.fork_pages(lengths, torch.full_like(lengths, -1), table, held, shared, pool, state, [], page=page,
                        blocks=blocks)
    return out, int(state[1]), blocks


def main():
    model = Model()
    prompts = [[5, 9, 2] * 20, [1, 2, 3, 4], [7] * 33]
    out, free, blocks = search(model, prompts, 12, 4, eos=3)
    for p, found in zip(prompts, out):
        print(f"prompt of {len(p)}:")
        for ids, score in found:
            print(f"  {score:9.4f}  {ids}")
    print(f"{free} of {blocks} pages free")


if __name__ == "__main__":
    main()
