"""Greedy decoding with drafted trees and a cache kept to a budget.

A small random decoder (torch products around the paged-cache operators of
rapidocrvl_b200.kvops) generates text for several sequences at once:

  1. drafts: the tokens that followed earlier occurrences of the last token, as a
     tree with one branch an occurrence (documents repeat themselves);
  2. one pass over the tree: tree_attention in every layer;
  3. the longest branch that greedy decoding would have taken is accepted, its keys
     and values go behind the cache with append (all layers at once);
  4. attention_mass adds up, for the accepted tokens, what each cached position
     received; a cache over the budget is cut with evict.

Without a budget the tokens equal those of one-token-at-a-time decoding: the
same calls with a tree of one token.

    python examples/tree_decode.py [--tokens 48] [--budget 64]
"""
import argparse
import math
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from rapidocrvl_b200 import kvops  # noqa: E402

VOCAB, HIDDEN, LAYERS, HEADS, KV_HEADS, DIM, PAGE = 96, 256, 2, 8, 2, 64, 16


class Decoder:
    """The weights, and one pass over flat tokens that are not in the cache yet."""

    def __init__(self, seed: int, device="cuda"):
        g = torch.Generator().manual_seed(seed)

        def w(*shape):
            return (torch.randn(*shape, generator=g) / math.sqrt(shape[-1])).to(device)

        self.embed, self.head = w(VOCAB, HIDDEN) * 8, w(VOCAB, HIDDEN)
        self.layers = [(w((HEADS + 2 * KV_HEADS) * DIM, HIDDEN), w(HIDDEN, HEADS * DIM), w(2 * HIDDEN, HIDDEN), w(HIDDEN, 2 * HIDDEN))
                       for _ in range(LAYERS)]
        self.freq = 1e4 ** (-torch.arange(0, DIM, 2, device=device) / DIM)

    def rotate(self, x, pos):
        a = pos[:, None, None] * self.freq
        c, s, (u, v) = a.cos(), a.sin(), x.chunk(2, -1)
        return torch.cat((u * c - v * s, v * c + u * s), -1)

    def __call__(self, ids, pos, cache, lens, indptr, mask):
        """Next-token logits, and of every layer the tokens' keys, values, queries and lse."""
        x, keys, values, queries, lses = self.embed[ids], [], [], [], []
        for layer, (qkv, o, up, down) in enumerate(self.layers):
            h = torch.nn.functional.rms_norm(x, (HIDDEN,)) @ qkv.T
            q, k, v = h.view(len(ids), -1, DIM).split((HEADS, KV_HEADS, KV_HEADS), 1)
            q, k, v = self.rotate(q, pos), self.rotate(k, pos), v.contiguous()
            out, lse = kvops.tree_attention(q, k, v, cache, lens, indptr, mask, layer=layer)
            x = x + out.flatten(1) @ o.T
            x = x + torch.nn.functional.silu(torch.nn.functional.rms_norm(x, (HIDDEN,)) @ up.T) @ down.T
            keys.append(k), values.append(v), queries.append(q), lses.append(lse)
        return torch.nn.functional.rms_norm(x, (HIDDEN,)) @ self.head.T, torch.stack(keys), torch.stack(values), queries, lses


def draft(tokens, width, depth):
    """A tree as (ids, parents), the last token its root: what followed the last
    token's most recent occurrences, a branch each."""
    ids, parents = [tokens[-1]], [-1]
    spots = [i for i in range(len(tokens) - 1) if tokens[i] == tokens[-1]]
    for i in spots[::-1][:width]:
        at = 0
        for t in tokens[i + 1:i + 1 + depth]:
            same = [n for n, p in enumerate(parents) if p == at and ids[n] == t]
            if not same:
                ids.append(t), parents.append(at)
            at = same[0] if same else len(ids) - 1
    return ids, parents


def ancestors(parents):
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
    return [m - (1 << 64) if m >> 63 else m for m in seen]


def generate(model, prompts, new, width=3, depth=4, budget=0):
    """Tokens of each prompt with at least `new` more, and the passes that took."""
    device, B = "cuda", len(prompts)
    room = -(-(max(map(len, prompts)) + new + depth + 1) // PAGE)
    pool = torch.zeros(B * room, LAYERS, KV_HEADS, 2, PAGE, DIM, device=device)
    table = torch.arange(B * room, dtype=torch.int32, device=device).view(B, room)
    cache = kvops.PagedCache(pool[:, :, :, 0], pool[:, :, :, 1], table)
    lens = torch.zeros(B, dtype=torch.int32, device=device)
    mass = torch.zeros(LAYERS, B, KV_HEADS, cache.capacity, device=device)

    def ints(x, dtype=torch.int32):
        return torch.tensor(x, dtype=dtype, device=device)

    # the prompts but their last tokens, one at a time (their rows see only what is before them)
    tokens = [list(p) for p in prompts]
    for i in range(max(map(len, prompts)) - 1):
        have = [i < len(p) - 1 for p in prompts]
        ids, pos = [p[i] for p, h in zip(prompts, have) if h], [i] * sum(have)
        indptr = ints([sum(have[:b]) for b in range(B + 1)])
        _, k, v, _, _ = model(ints(ids, torch.long), ints(pos), cache, lens, indptr, ints([1] * len(ids), torch.int64))
        lens = kvops.append(cache, k, v, lens, indptr)
    passes = 0
    while min(len(t) - len(p) for t, p in zip(tokens, prompts)) < new:
        # a sequence that is done drafts nothing
        trees = [draft(t, width, depth) if len(t) - len(p) < new else ([], []) for t, p in zip(tokens, prompts)]
        starts = [0]
        for ids, _ in trees:
            starts.append(starts[-1] + len(ids))
        depths = []
        for (ids, parents), t in zip(trees, tokens):
            d = []
            for p in parents:
                d.append(d[p] + 1 if p >= 0 else 0)
            depths += [len(t) - 1 + x for x in d]
        indptr = ints(starts)
        logits, k, v, qs, lses = model(ints([i for ids, _ in trees for i in ids], torch.long), ints(depths), cache, lens, indptr,
                                       ints([m for _, parents in trees for m in ancestors(parents)], torch.int64))
        passes += 1
        best = logits.argmax(-1).tolist()
        paths, counted = [], []
        for b, (ids, parents) in enumerate(trees):
            path = [0] if ids else []  # the root is always taken; a child while it is what greedy decoding says
            while path:
                want = best[starts[b] + path[-1]]
                child = [n for n, p in enumerate(parents) if p == path[-1] and ids[n] == want]
                tokens[b].append(want)
                if not child:
                    break
                path.append(child[0])
            paths.append(path), counted.append(sum(1 << n for n in path))
        for layer in range(LAYERS):
            kvops.attention_mass(qs[layer], lses[layer], cache, lens, indptr, layer=layer, counted=ints(counted, torch.int64),
                                 acc=mass[layer], out=mass[layer])
        most = max(map(len, paths))
        lens = kvops.append(cache, k, v, lens, indptr, path=ints([p + [0] * (most - len(p)) for p in paths]),
                            n_path=ints([len(p) for p in paths]))
        if budget and int(lens.max()) > budget:
            _, kept, lens = kvops.evict(cache, mass, lens, keep=budget * 3 // 4, sinks=4, recent=budget // 4)
            mass.zero_()
            mass[..., :kept.shape[-1]] = kept
    return tokens, passes, lens.tolist()


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--tokens", type=int, default=48)
    ap.add_argument("--budget", type=int, default=64)
    a = ap.parse_args()
    model = Decoder(0)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in (5, 17, 40)]
    plain, steps, _ = generate(model, prompts, a.tokens, width=0)
    tree, passes, lens = generate(model, prompts, a.tokens)
    for p, x, y in zip(prompts, plain, tree):
        n = len(p) + a.tokens
        if x[:n] != y[:n]:
            raise SystemExit(f"the tree changed the tokens: {x[len(p):n]} / {y[len(p):n]}")
    print(f"{len(prompts)} sequences, {a.tokens} tokens each: {steps} passes of one token, {passes} with trees, the same tokens; caches {lens}")
    cut, passes, lens = generate(model, prompts, a.tokens, budget=a.budget)
    assert max(lens) <= a.budget + 8
    print(f"with caches cut to at most {a.budget}: {passes} passes, caches {lens}")


if __name__ == "__main__":
    main()
