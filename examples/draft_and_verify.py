"""Generation with drafted trees over a paged int8 cache, with the four paged-cache operators.

    python examples/draft_and_verify.py [--steps N] [--batch B] [--temperature T]

A step drafts a tree of tokens after each sequence's last one, writes the nodes' keys and values into
the cache (cache_write), lets all nodes attend to the context and to their ancestors (tree_attention),
holds the drafts against the target's logits (verify_drafts) and moves the taken branch's rows next to
the context (cache_read, cache_write).  The target is one attention layer with random weights, the
drafter its first guesses without the attention: a stand-in for models, with every operator used as a
serving loop uses it.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "t4a-cuda-kernels_b200"))
import t4a_b200 as t4  # noqa: E402

BRANCHES = 2  # children of a drafted node


class Target:
    """One layer of attention between an embedding and its transpose."""

    def __init__(self, vocab=4096, heads=8, kv_heads=2, dim=64, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.vocab, self.heads, self.kv_heads, self.dim = vocab, heads, kv_heads, dim
        width = heads * dim

        def weight(*shape):
            return (torch.randn(shape, generator=gen, device="cuda") * shape[0] ** -0.5).to(torch.bfloat16)

        self.embedding = torch.randn(vocab, width, generator=gen, device="cuda").to(torch.bfloat16)
        self.q, self.k, self.v = weight(width, width), weight(width, kv_heads * dim), weight(width, kv_heads * dim)
        self.mix = weight(width, width)

    def rows(self, tokens):
        """(x, q, key, value) of tokens [...]."""
        x = self.embedding[tokens]
        shape = tokens.shape
        return (x, (x @ self.q).view(*shape, self.heads, self.dim), (x @ self.k).view(*shape, self.kv_heads, self.dim),
                (x @ self.v).view(*shape, self.kv_heads, self.dim))

    def logits(self, x, attended):
        return ((x @ self.mix + 0.3 * attended.flatten(-2)) @ self.embedding.t()).float() / 4

    def guesses(self, tokens, count):
        """The likeliest followers without the context."""
        return ((self.embedding[tokens] @ self.mix) @ self.embedding.t()).topk(count, dim=-1).indices


class Cache:
    """Pages of int8 rows with their scales; sequence b's place p lies in page table[b, p // page]."""

    def __init__(self, batch, places, kv_heads, dim, page=16):
        self.page = page
        width = -(-places // page)
        shape = (batch * width, page, kv_heads, dim)
        self.k, self.v = (torch.zeros(shape, dtype=torch.int8, device="cuda") for _ in range(2))
        self.scales = {name: torch.zeros(shape[:3], device="cuda") for name in ("k_scale", "v_scale")}
        self.table = torch.randperm(batch * width, device="cuda").view(batch, width).int()

    def slots(self, places):
        """Of places [batch, n]."""
        return (self.table.long().gather(1, places // self.page) * self.page + places % self.page).flatten()

    def write(self, key, value, places):
        t4.cache_write(key.flatten(0, 1), value.flatten(0, 1), self.k, self.v, self.slots(places), **self.scales)

    def move(self, old, new):
        """Rows from places `old` to places `new`; 32-bit values give the same codes again."""
        key, value = t4.cache_read(self.k, self.v, self.slots(old), torch.float32, **self.scales)
        t4.cache_write(key, value, self.k, self.v, self.slots(new), **self.scales)


def tree(depth):
    """(parents, which nodes a node sees) of a root and `depth` levels below it, the first child of a level
    going on."""
    parents, last = [-1], 0
    for _ in range(depth):
        first = len(parents)
        parents += [last] * BRANCHES
        last = first
    sees = torch.eye(len(parents), dtype=torch.bool)
    for i, parent in enumerate(parents):
        if parent >= 0:
            sees[i] |= sees[parent]
    return parents, sees


def generate(target, prompt, count, depth=3, temperature=0.0, seed=1):
    """At least `count` tokens after each prompt [batch, n], and the steps that they took; depth 0 drafts
    nothing: a token a step.  A sequence that has its tokens waits for the others: its step is repeated."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    batch, n = prompt.shape
    parents, sees = tree(depth)
    nodes = len(parents)
    cache = Cache(batch, n + count + (depth + 1) + nodes, target.kv_heads, target.dim)
    parents_of = torch.tensor(parents, dtype=torch.int32, device="cuda").expand(batch, nodes).contiguous()
    sees = sees.cuda().expand(batch, nodes, nodes)
    offsets = torch.arange(nodes, device="cuda")
    # All of the prompt but its last token, the first root.
    _, _, key, value = target.rows(prompt[:, :-1])
    cache.write(key, value, torch.arange(n - 1, device="cuda").expand(batch, n - 1))
    context = torch.full((batch,), n - 1, dtype=torch.int32, device="cuda")
    tokens = torch.zeros(batch, nodes, dtype=torch.int32, device="cuda")
    tokens[:, 0] = prompt[:, -1]
    out, steps = [[] for _ in range(batch)], 0
    while min(len(o) for o in out) < count:
        level, at = tokens[:, 0].long(), 1
        for _ in range(depth):
            guesses = target.guesses(level, BRANCHES)
            tokens[:, at:at + BRANCHES] = guesses
            level, at = guesses[:, 0], at + BRANCHES
        x, q, key, value = target.rows(tokens.long())
        cache.write(key, value, context[:, None].long() + offsets)
        attended, _ = t4.tree_attention(q, cache.k, cache.v, cache.table, context, mask=sees, **cache.scales)
        logits = target.logits(x, attended)
        uniforms = torch.rand(batch, nodes, generator=gen, device="cuda")
        race = torch.empty(batch, target.vocab, device="cuda").exponential_(generator=gen).clamp_min_(1e-30).reciprocal_()
        taken, path, said, _ = t4.verify_drafts(logits, tokens, parents_of, uniforms=uniforms, race=race,
                                                temperature=temperature)
        if depth:
            # The branch's rows follow the root's; places that no node was taken for move onto themselves.
            kept = path[:, :depth].long()
            new = offsets[1:depth + 1].expand(batch, depth)
            old = torch.where(kept >= 0, kept, new)
            cache.move(context[:, None].long() + old, context[:, None].long() + new)
        steps += 1
        goes_on = torch.tensor([len(o) < count for o in out], device="cuda")
        for o, row, k in zip(out, said.tolist(), taken.tolist()):
            if len(o) < count:
                o.extend(row[:k + 1])
        context += torch.where(goes_on, taken + 1, 0)
        tokens[:, 0] = torch.where(goes_on, said.gather(1, taken[:, None].long())[:, 0], tokens[:, 0])
    return out, steps


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=64, help="tokens to generate")
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--temperature", type=float, default=0.0)
    args = ap.parse_args()
    target = Target()
    prompt = torch.randint(0, target.vocab, (args.batch, 100), device="cuda")
    out, steps = generate(target, prompt, args.steps, temperature=args.temperature)
    said = sum(len(o) for o in out)
    print(f"{said} tokens of {args.batch} sequences in {steps} steps: {said / args.batch / steps:.2f} tokens a step")


if __name__ == "__main__":
    main()
