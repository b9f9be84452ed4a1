"""Speculative decoding with drafted trees: the step's operators in one loop.

A small random transformer generates for a batch of requests.  A prompt is
ingested as a causal chunk; then every step drafts a tree of seven nodes per
request, runs the target model once over all nodes, draws the target's token
at each of them, and keeps the accepted path:

  plan_blocks -> per layer (rotary with cache writes -> tree_attention)
  -> vocab_head -> sample_rows -> commit_tree

Lengths, block tables, page pool and pending tokens stay on the device.  Greedy
output is that of decoding one token at a time (``drafts=False``).  Requests that
find the pool short wait for pages that others give back at their end.

    python examples/tree_decode.py
"""
import os
import sys
from dataclasses import dataclass, field

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from deepseekrpc_amd import batch, tree  # noqa: E402

# Root, two children, two children each.
PARENTS = (-1, 0, 0, 1, 1, 2, 2)


class Model:
    """Random weights: pre-norm attention and a gated product, grouped heads."""

    def __init__(self, vocab=512, dim=256, layers=2, heads=4, kv=2, seed=0, device="cuda"):
        g = torch.Generator(device="cpu").manual_seed(seed)
        self.vocab, self.dim, self.layers, self.heads, self.kv, self.head = vocab, dim, layers, heads, kv, dim // heads
        self.device = device

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=g) * cols ** -0.5).to(device, torch.bfloat16)

        self.embed = torch.randn(vocab, dim, generator=g).to(device, torch.bfloat16)
        self.qkv = [weight(dim + 2 * kv * self.head, dim) for _ in range(layers)]
        self.out = [weight(dim, dim) for _ in range(layers)]
        self.up = [weight(4 * dim, dim) for _ in range(layers)]
        self.down = [weight(dim, 2 * dim) for _ in range(layers)]
        # A sharp head that leans on the input token's own direction.
        self.lm_head = (4 * weight(vocab, dim) + torch.roll(self.embed, -1, 0)).contiguous()
        self.freqs, self.magnitude = tree.rotary_frequencies(self.head, scaling="ramp", factor=4.0, original=256,
                                                             device=device)

    @staticmethod
    def norm(x):
        x = x.float()
        return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).to(torch.bfloat16)

    def forward(self, tokens, plan, k_caches, v_caches, attend=tree.tree_attention):
        """Hidden states of the step's tokens; their keys and values go to the caches."""
        x = self.embed[tokens]
        n, split = tokens.numel(), [self.dim, self.kv * self.head, self.kv * self.head]
        for i in range(self.layers):
            q, k, v = (self.norm(x) @ self.qkv[i].t()).split(split, -1)
            q, k, v = (t.view(n, -1, self.head) for t in (q, k, v))
            q = tree.rotary(q, k, plan.positions, self.freqs, v=v, magnitude=self.magnitude, slots=plan.slots,
                            k_cache=k_caches[i], v_cache=v_caches[i]).q
            out = attend(q, k_caches[i], v_caches[i], plan.table, plan.offsets, plan.kv_lengths,
                         visible=plan.visible).out
            x = x + out.view(n, -1) @ self.out[i].t()
            a, b = (self.norm(x) @ self.up[i].t()).chunk(2, -1)
            x = x + (torch.nn.functional.silu(a) * b) @ self.down[i].t()
        return self.norm(x)

    def logits(self, hidden):
        return torch.cat([batch.vocab_head(h.contiguous(), self.lm_head, records=False).logits
                          for h in hidden.split(256)])


@dataclass
class Output:
    ids: list = field(default_factory=list)
    steps: int = 0
    waits: int = 0  # steps without pages for it
    free_pages: int = 0


def generate(model, prompts, new_tokens, *, drafts=True, page=16, policy=None, uniforms=None, missing=0):
    """``new_tokens`` ids for each prompt (lists of token ids).  ``policy`` and
    ``uniforms(step, rows)`` make it sample; without them it is greedy.  The pool
    is ``missing`` pages short of what all requests could hold together: fewer
    than there are requests, so that some request always finds its pages."""
    dev, R = model.device, len(prompts)
    longest = max(map(len, prompts)) + new_tokens + len(PARENTS)
    width = -(-longest // page)
    blocks = sum(-(-(len(p) + new_tokens + len(PARENTS)) // page) for p in prompts) - missing
    shape = (blocks, page, model.kv, model.head)
    k_caches = [torch.zeros(shape, dtype=torch.bfloat16, device=dev) for _ in range(model.layers)]
    v_caches = [torch.zeros_like(t) for t in k_caches]
    table = torch.full((R, width), -1, dtype=torch.int32, device=dev)
    pool, state = tree.page_pool(blocks, dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    held, lengths = i32([0] * R), i32([0] * R)
    policy = dict(temperature=0.0) if policy is None else policy

    def draw(logits, step):
        rows = logits.shape[0]
        u = None if uniforms is None else uniforms(step, rows)
        if u is None:  # greedy rows use no draw, but ask for one to be offered
            u = torch.zeros(rows, dtype=torch.float64, device=dev)
        return batch.sample_rows(logits, [policy] * rows, uniforms=u).tokens

    # Each token's two likeliest successors after itself alone: the draft.
    everything = torch.arange(model.vocab, device=dev)
    draft = model.logits(model.norm(model.embed[everything])).topk(2).indices.to(torch.int32)

    # Prompts, as one causal chunk.
    flat = i32([t for p in prompts for t in p])
    plan = tree.plan_blocks(lengths, i32([len(p) for p in prompts]), table, held, pool, state, blocks=blocks,
                            page=page, capacity=flat.numel())
    hidden = model.forward(flat, plan, k_caches, v_caches)
    assert not bool(plan.status.any())  # the pool holds all prompts
    pending = draw(model.logits(hidden[plan.offsets[1:].long() - 1]), 0)
    lengths = plan.kv_lengths
    left = torch.full((R,), new_tokens - 1, dtype=torch.int32, device=dev)
    result = [Output([t]) for t in pending.tolist()]

    nodes = len(PARENTS) if drafts else 1
    parents = i32(PARENTS[:nodes]).repeat(R)
    step = 0
    while int(left.max()) > 0:
        step += 1
        busy = left > 0
        # Requests that are done end, and give their pages back.
        added = torch.where(busy, nodes, torch.where(held > 0, -1, 0)).to(torch.int32)
        plan = tree.plan_blocks(lengths, added, table, held, pool, state, blocks=blocks, page=page,
                                capacity=R * nodes, parents=parents)
        trees = [pending.clamp(min=0)]
        for node in range(1, nodes):  # children of one node take its successors in order
            of = PARENTS[node]
            trees.append(draft[trees[of].long(), PARENTS[:node].count(of)])
        owner = plan.owners.clamp(min=0).long()
        local = torch.arange(R * nodes, device=dev) - plan.offsets[owner]
        tokens = torch.stack(trees, 1)[owner, local.clamp(0, nodes - 1)]
        logits = model.logits(model.forward(tokens, plan, k_caches, v_caches))
        done = tree.commit_tree(parents, tokens, draw(logits, step), plan.offsets, plan.kv_lengths, table,
                                k_caches + v_caches, output_limit=left, lengths=lengths, pending=pending,
                                plan_status=plan.status)
        # A request that lacks pages is served when there are some.
        assert bool(((done.status == 0) | (done.status == tree.E_BLOCKS)).all())
        lengths, pending, left = done.lengths, done.pending, left - done.count
        for r, (n, row, status) in enumerate(zip(done.count.tolist(), done.ids.tolist(), done.status.tolist())):
            result[r].ids += row[:n]
            result[r].steps += n > 0
            result[r].waits += status == tree.E_BLOCKS
    # The others end.
    tree.plan_blocks(lengths, i32([-1] * R), table, held, pool, state, blocks=blocks, page=page, capacity=1)
    for o in result:
        o.free_pages = int(state[1])
    assert int(state[1]) == blocks
    return result


def main():
    model = Model()
    prompts = [list(range(7, 7 + n)) for n in (5, 1, 40, 17)]
    one = generate(model, prompts, 48, drafts=False)
    many = generate(model, prompts, 48)
    for a, b in zip(one, many):
        print(f"{len(b.ids)} ids in {b.steps} steps ({len(b.ids) / max(1, b.steps):.2f} a step), "
              f"same as one at a time: {a.ids == b.ids}")


if __name__ == "__main__":
    main()
