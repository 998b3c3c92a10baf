"""Retrieve passages, keep their keys and values in 4 bits, generate tokens that attend to them.

    PYTHONPATH=. python examples/answer_from_retrieved.py [--layers 2] [--tokens 8]

A corpus of passages is searched with the compressed MaxSim scan; the tokens of the best passages are run through a
small decoder (random weights in 4 bits) as one prompt chunk per query, and tokens are generated one at a time over
the cache.  Everything after the search stays on the GPU.
"""

import argparse

import numpy as np
import torch

import maxsim_b200 as m


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

    def __call__(self, x, slots, page_table, lengths, query_offsets, most):
        """``x`` ``[rows, dim]``: the rows' keys and values go to ``slots``, then they attend to their sequences."""
        qkv = self.qkv(_norm(x)).unflatten(1, (self.heads + 2 * self.kv_heads, self.head_dim))
        query, keys, values = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=1)
        self.cache.append(keys, values, slots)
        seen = self.cache.attend(query, page_table, lengths, query_offsets=query_offsets, max_query_tokens=most)
        x = x + self.out(seen.flatten(1))
        return x + self.down(torch.nn.functional.silu(self.up(_norm(x))))


def _norm(x):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(dim=-1, keepdim=True) + 1e-6)).to(x.dtype)


def main(layers=2, tokens=8, queries=3, passages=200, k=2, dim=128, heads=8, kv_heads=2, head_dim=64, page_size=16,
         vocabulary=1000, seed=0):
    rng = np.random.default_rng(seed)
    generator = torch.Generator(device="cuda").manual_seed(seed)

    # 1. Search: passages of 20 to 60 token vectors; each query is a noisy piece of one of them.
    lengths = rng.integers(20, 61, passages)
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    vectors = rng.standard_normal((offsets[-1], dim)).astype(np.float32)
    vectors /= np.linalg.norm(vectors, axis=1, keepdims=True)
    wanted = rng.choice(passages, queries, replace=False)
    query = np.stack([vectors[offsets[w]:offsets[w] + 16] for w in wanted])
    query += 0.05 * rng.standard_normal(query.shape).astype(np.float32)
    index = m.Index.from_embeddings([f"passage {i}" for i in range(passages)], vectors, offsets, mode="int4_per_token")
    _, found = m.Reranker(index, device="cuda", int4_query="int8").search_arrays(query, k=k)

    # 2. The prompt of a query: the tokens of the passages found for it, one after the other, in pages of its own.
    prompts = [np.concatenate([vectors[offsets[d]:offsets[d + 1]] for d in row]) for row in found]
    sizes = np.array([len(p) for p in prompts])
    per = int(-(-(sizes.max() + tokens) // page_size))
    page_table = torch.randperm(queries * per, generator=generator, device="cuda").to(torch.int32).view(queries, per)
    model = [Layer(dim, heads, kv_heads, head_dim, queries * per, page_size, generator) for _ in range(layers)]
    words = torch.randn((vocabulary, dim), generator=generator, device="cuda", dtype=torch.float32).to(torch.bfloat16)
    unembed = m.Int4Linear.from_weight(words, group_size=64)

    def forward(x, sequence, position, length, query_offsets, most):
        slots = model[0].cache.slots(page_table, sequence, position)
        for layer in model:
            x = layer(x, slots, page_table, length, query_offsets, most)
        return x

    x = torch.from_numpy(np.concatenate(prompts)).cuda().to(torch.bfloat16) * dim**0.5
    sequence = torch.repeat_interleave(torch.arange(queries), torch.from_numpy(sizes)).cuda()
    position = torch.cat([torch.arange(n) for n in sizes]).cuda()
    length = torch.from_numpy(sizes).to(torch.int32).cuda()
    starts = torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)])).to(torch.int32).cuda()
    x = forward(x, sequence, position, length, starts, int(sizes.max()))

    # 3. Generate: the last row of each sequence gives the next token, one row per sequence from here on.
    last = x[starts[1:].long() - 1]
    everyone, answer = torch.arange(queries, device="cuda"), []
    for _ in range(tokens):
        token = unembed(_norm(last)).float().argmax(dim=1)
        answer.append(token)
        last = forward(words[token], everyone, length.long(), length + 1, None, None)
        length += 1
    return wanted, found, torch.stack(answer, dim=1)


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--layers", type=int, default=2)
    parser.add_argument("--tokens", type=int, default=8)
    args = parser.parse_args()
    wanted, found, answer = main(layers=args.layers, tokens=args.tokens)
    for w, row, tokens in zip(wanted, found, answer.tolist()):
        print(f"passage {w}: found {row.tolist()}, generated {tokens}")
