"""Generate from a 4-bit cache by drafted trees: several tokens a step, one pass over the model each.

    PYTHONPATH=. python examples/answer_with_drafts.py [--tokens 24] [--window 64 --sinks 4]

A small decoder (random weights in 4 bits, rotary positions) reads prompts of different lengths.  Each step drafts a tree
of five tokens for every sequence (the next token, which is known, the runner-up, and guesses of what follows from the
words alone), runs all nodes through the model at once, keeps the path that the model itself would have taken, moves its
keys and values to the places after the context, and gives the rest of the pages back.  Nothing waits for the GPU until the
end.
"""

import argparse

import torch

import maxsim_b200 as m

# A step's tree: two candidates, a child of each, and a grandchild of the first.
PARENTS = [-1, -1, 0, 1, 2]
PATH = [0, 2, 4]  # the nodes that can be accepted one after the other


class Layer:
    """Attention and a two-layer perceptron; all products with 4-bit weights, keys and values in a 4-bit cache."""

    def __init__(self, dim, heads, kv_heads, head_dim, pages, page_size, generator):
        def linear(n, k):
            w = torch.randn((n, k), generator=generator, device="cuda") * k**-0.5
            return m.Int4Linear.from_weight(w, group_size=64)

        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.qkv = linear((heads + 2 * kv_heads) * head_dim, dim)
        self.out = linear(dim, heads * head_dim)
        self.up, self.down = linear(4 * dim, dim), linear(dim, 4 * dim)
        self.cache = m.Int4KVCache(pages, page_size, kv_heads, head_dim)

    def __call__(self, x, rotary, positions, slots, table, offsets, most, **mask):
        qkv = self.qkv(_norm(x)).unflatten(1, (self.heads + 2 * self.kv_heads, self.head_dim))
        query, keys, values = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=1)
        rotary(query, keys, positions, out=(query, keys))
        self.cache.append(keys, values, slots)
        seen = self.cache.attend(query, table.page_table, table.lengths, query_offsets=offsets, max_query_tokens=most, **mask)
        x = x + self.out(seen.flatten(1))
        return x + self.down(torch.nn.functional.silu(self.up(_norm(x))))


def _norm(x):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(dim=-1, keepdim=True) + 1e-6)).to(x.dtype)


def main(prompts=(37, 5, 80), tokens=24, layers=2, dim=128, heads=8, kv_heads=2, head_dim=64, page_size=16, vocabulary=1000,
         window=None, sinks=0, seed=0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    batch, nodes = len(prompts), len(PARENTS)
    per = -(-(max(prompts) + len(PATH) * tokens + nodes) // page_size)
    model = [Layer(dim, heads, kv_heads, head_dim, batch * per, page_size, generator) for _ in range(layers)]
    table = m.PageTable(batch * per, page_size, batch, per)
    rotary = m.Rotary(head_dim)
    words = torch.randn((vocabulary, dim), generator=generator, device="cuda").to(torch.bfloat16)
    unembed = m.Int4Linear.from_weight(torch.randn((vocabulary, dim), generator=generator, device="cuda"), group_size=64)
    mask = {"window": window, "sinks": sinks}

    def forward(token, positions, slots, offsets, most, **more):
        x = words[token]
        for layer in model:
            x = layer(x, rotary, positions, slots, table, offsets, most, **mask, **more)
        return unembed(_norm(x)).float()

    # The prompts, all in one call; the last row of each gives its first two candidates.
    sizes = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    text = torch.randint(vocabulary, (sum(prompts),), generator=generator, device="cuda")
    offsets, slots, positions = table.extend(sizes, sum(prompts))
    logits = forward(text, positions, slots, offsets, max(prompts))[offsets[1:].long() - 1]

    grow = torch.full((batch,), nodes, dtype=torch.int32, device="cuda")
    parents = torch.tensor(PARENTS * batch, dtype=torch.int32, device="cuda")
    first = torch.arange(batch, device="cuda").unsqueeze(1) * nodes  # each sequence's first row
    place, path = torch.arange(len(PATH), device="cuda"), torch.tensor(PATH, device="cuda")
    answer, counts = [], []
    for _ in range(tokens):
        before = table.lengths.clone()
        draft = torch.empty((batch, nodes), dtype=torch.int64, device="cuda")
        draft[:, :2] = logits.topk(2, dim=1).indices
        guess = unembed(words[draft[:, :2].flatten()]).float().argmax(dim=1)
        draft[:, 2:4] = guess.view(batch, 2)
        draft[:, 4] = unembed(words[draft[:, 2]]).float().argmax(dim=1)
        offsets, slots, _ = table.extend(grow, batch * nodes)
        ancestors, depths = m.draft_ancestors(parents, offsets, max_query_tokens=nodes)
        positions = before.repeat_interleave(nodes) + depths
        logits = forward(draft.flatten(), positions, slots, offsets, nodes, ancestors=ancestors).view(batch, nodes, -1)
        # The first candidate is the model's own; a node below it is, where the model takes its word after the parent.
        says = logits.argmax(dim=2)
        right = torch.stack((says[:, 0] == draft[:, 2], says[:, 2] == draft[:, 4]), dim=1)
        count = 1 + right.int().cumprod(dim=1).sum(dim=1)
        kept = place < count.unsqueeze(1)
        source = torch.where(kept, slots[first + path], -1)
        for layer in model:
            layer.cache.move(source.flatten(), slots[first + place].flatten())
        table.truncate(before + count.int())
        answer.append(torch.where(kept, draft[:, path], -1))
        counts.append(count)
        logits = logits[torch.arange(batch, device="cuda"), path[count - 1]]
    return torch.stack(answer, dim=1), torch.stack(counts, dim=1)


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--tokens", type=int, default=24)
    parser.add_argument("--window", type=int, default=None)
    parser.add_argument("--sinks", type=int, default=0)
    args = parser.parse_args()
    answer, counts = main(tokens=args.tokens, window=args.window, sinks=args.sinks)
    for row, n in zip(answer.flatten(1).tolist(), counts.sum(dim=1).tolist()):
        print(f"{n} tokens in {args.tokens} steps: {[t for t in row if t >= 0]}")
