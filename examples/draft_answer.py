"""Answering with drafted tokens: a model in 8-bit integers with a paged cache, whose next tokens are proposed by a cheap model and checked several at a time.

    python examples/draft_answer.py [--sequences 4] [--prompt 200] [--answer 64] [--hidden 1024] [--layers 4] [--heads 16] [--shared 4] [--vocab 4000] [--nodes 12]

Random weights of a small model.  All products are 8-bit (`verinf_amd.prover.inference`); positions, cache, attention and the trees of drafts are
`verinf_amd.prover.generation`'s.  The draft model is the model without its layers: what a token's embedding alone says of the next.  Tokens come out distributed
as the model's own whatever the drafts are; how many of them are accepted says how good the drafts were.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from verinf_amd.prover import generation as gen  # noqa: E402
from verinf_amd.prover import inference as inf  # noqa: E402


class Model:
    def __init__(self, hidden=1024, layers=4, heads=16, shared=4, dim=64, vocab=4000, seed=0, cache_type=torch.int8):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weights(n, k, size=1.0):
            return inf.quantize_rows(torch.randn((n, k), generator=g, device="cuda") * (size / k ** 0.5))

        self.heads, self.shared, self.dim, self.layers, self.cache_type, self.vocab = heads, shared, dim, layers, cache_type, vocab
        self.embedding = torch.randn((vocab, hidden), generator=g, device="cuda")
        self.plan = gen.rotary_plan(dim)
        self.blocks = [{"qkv": weights((heads + 2 * shared) * dim, hidden), "out": weights(hidden, heads * dim, 0.3), "gate": weights(2 * hidden, hidden),
                        "up": weights(2 * hidden, hidden), "down": weights(hidden, 2 * hidden, 0.3)} for _ in range(layers)]
        self.head = weights(vocab, hidden, 3.0)

    def caches(self, pages, page_size):
        """All layers' heads of a page lie together, so that one call moves a path's entries in all of them."""
        shape = (pages, 2, self.layers * self.shared, page_size, self.dim)
        both = torch.zeros(shape, dtype=self.cache_type, device="cuda")
        scales = torch.zeros(shape[:4], device="cuda") if self.cache_type == torch.int8 else None

        def of(first, count):
            heads = slice(first * self.shared, (first + count) * self.shared)
            return gen.Cache(both[:, 0, heads], both[:, 1, heads], *(() if scales is None else (scales[:, 0, heads], scales[:, 1, heads])))

        return of(0, self.layers), [of(i, 1) for i in range(self.layers)]

    @staticmethod
    def product(x, w, dtype=torch.bfloat16):
        q, s = inf.quantize_rows(x)
        return inf.int8_matmul(q, w[0], s, w[1], dtype=dtype)

    @staticmethod
    def norm(x):
        return x * torch.rsqrt(x.square().mean(dim=1, keepdim=True) + 1e-6)

    def logits(self, x):
        return self.product(self.norm(x), self.head, torch.float32)

    def draft_logits(self, tokens):
        return self.logits(self.embedding[tokens])

    def forward(self, tokens, positions, caches, batch, parents=None, longest=None):
        """Logits behind each of the new tokens, whose keys and values go into the caches."""
        x, n = self.embedding[tokens], tokens.shape[0]
        for block, cache in zip(self.blocks, caches):
            qkv = self.product(self.norm(x), block["qkv"]).view(n, -1, self.dim)
            q, k, v = qkv.split((self.heads, self.shared, self.shared), dim=1)
            gen.append_tokens(cache, k, v, batch, positions, self.plan)
            o = gen.attend_cache(gen.rotate_heads(q, positions, self.plan), cache, batch, parents, longest=longest)
            x = x + self.product(o.view(n, -1), block["out"], torch.float32)
            a, s = inf.quantize_rows(self.norm(x))
            h = inf.int8_gated(a, block["gate"][0], block["up"][0], s, block["gate"][1], block["up"][1])
            x = x + self.product(h, block["down"], torch.float32)
        return self.logits(x)


def draw_trees(model, roots, nodes, g):
    """A tree for each root, drawn from the draft model: every node has three children, in the order of the nodes, until there are enough.
    Returns tokens, parents, depths (each sequences * nodes) and the draft's logits behind every node."""
    b = roots.shape[0]
    parent = [-1] + [(i - 1) // 3 for i in range(1, nodes)]
    depth = [0] * nodes
    for i in range(1, nodes):
        depth[i] = depth[parent[i]] + 1
    tokens = torch.zeros((b, nodes), dtype=torch.int64, device="cuda")
    tokens[:, 0] = roots
    logits = torch.zeros((b, nodes, model.vocab), device="cuda")
    for i in range(nodes):
        logits[:, i] = model.draft_logits(tokens[:, i])
        children = [c for c in range(1, nodes) if parent[c] == i]
        if children:
            tokens[:, children] = torch.multinomial(torch.softmax(logits[:, i], dim=1), len(children), replacement=True, generator=g)
    parents = torch.tensor(parent, dtype=torch.int32, device="cuda").repeat(b)
    return tokens.flatten(), parents, torch.tensor(depth, device="cuda").repeat(b), logits.view(b * nodes, -1), max(depth)


def answer(model, prompts, length, nodes=12, page_size=16, seed=0):
    """`length` tokens at least behind each of the prompts (sequences, prompt): lists of tokens, and the steps that they took."""
    b, n = prompts.shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    longest = n + length + 2 * nodes
    width = -(-longest // page_size)
    layers, caches = model.caches(b * width, page_size)
    pages = torch.randperm(b * width, generator=g, device="cuda").view(b, width).int()
    # the prompts but for their last tokens, which are the first trees' roots
    starts = torch.arange(b + 1, device="cuda", dtype=torch.int32)
    lengths = torch.full((b,), n - 1, dtype=torch.int32, device="cuda")
    batch = gen.Batch(starts * (n - 1), lengths, pages)
    model.forward(prompts[:, :-1].reshape(-1), torch.arange(n - 1, device="cuda").repeat(b), caches, batch, longest=longest)
    root, out, steps = prompts[:, -1], [[] for _ in range(b)], 0
    while min(len(o) for o in out) < length:
        tokens, parents, depths, drafted, deepest = draw_trees(model, root, nodes, g)
        positions = (lengths.long()[:, None] + depths.view(b, nodes)).flatten()
        batch = gen.Batch(starts * nodes, lengths + nodes, pages)
        logits = model.forward(tokens, positions, caches, batch, parents, longest)
        uniforms = torch.rand(b * nodes, generator=g, device="cuda", dtype=torch.float64)
        counts, path, said = gen.verify_drafts(logits, tokens, starts * nodes, parents, uniforms, deepest, drafted)
        lengths = gen.keep_drafts(layers, batch, path, counts)         # the root and the path; what was said last is the next root
        root = said.gather(1, counts[:, None])[:, 0]
        for o, row in zip(out, said.tolist()):
            o += [t for t in row if t >= 0]
        steps += 1
        if max(len(o) for o in out) > length + nodes:                  # where the fastest has no pages left
            break
    return out, steps


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("sequences", 4), ("prompt", 200), ("answer", 64), ("hidden", 1024), ("layers", 4), ("heads", 16), ("shared", 4), ("vocab", 4000), ("nodes", 12), ("seed", 0)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    model = Model(a.hidden, a.layers, a.heads, a.shared, 64, a.vocab, a.seed)
    prompts = torch.randint(0, a.vocab, (a.sequences, a.prompt), generator=torch.Generator().manual_seed(a.seed)).cuda()
    answer(model, prompts, 4, a.nodes)           # every kernel has been loaded before the time is taken
    torch.cuda.synchronize()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    out, steps = answer(model, prompts, a.answer, a.nodes)
    end.record()
    torch.cuda.synchronize()
    total = sum(len(o) for o in out)
    print(f"{total} tokens of {a.sequences} answers in {steps} steps, {total / steps / a.sequences:.2f} a step and answer, {start.elapsed_time(end) / steps:.2f} ms a step")
    return 0


if __name__ == "__main__":
    sys.exit(main())
