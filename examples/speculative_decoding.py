"""Speculative decoding over a paged K/V cache with scree_b200.

A small decoder with random weights answers a batch of prompts of different
lengths.  Each step drafts a tree of tokens per sequence, runs the model once
over all trees (attention over the cache with the trees' visibility), keeps the
path that greedy decoding would have taken, scores it, and gives the rest of
the draft back.  The tokens are those of decoding one at a time.

    python examples/speculative_decoding.py
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

if str(Path(__file__).resolve().parent.parent) not in sys.path:
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import scree_b200 as scree
from scree_b200 import _lib, paged
from scree_b200.kernels.native import rmsnorm_qkv, token_logprobs, varlen_rmsnorm_triton

WIDTH, HEADS, KV_HEADS, DIM, LAYERS, VOCAB = 512, 8, 2, 64, 2, 1024
PAGE = 16


class Decoder:
    """Pre-norm attention and MLP blocks; the K/V of every token lives in a paged cache."""

    def __init__(self, device, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)

        def w(*shape):
            return (torch.randn(shape, generator=g, device=device) / shape[0] ** 0.5).to(torch.bfloat16)

        self.embed = w(VOCAB, WIDTH) * VOCAB**0.5
        self.head = w(WIDTH, VOCAB)
        self.layers = [dict(qkv=w(WIDTH, (HEADS + 2 * KV_HEADS) * DIM), out=w(HEADS * DIM, WIDTH),
                            up=w(WIDTH, 2 * WIDTH), down=w(2 * WIDTH, WIDTH)) for _ in range(LAYERS)]

    def __call__(self, tokens, cache, slots, mask=None):
        """Logits of packed new tokens (an Array of ids).  Room for them is reserved in the
        cache; their K/V is written here, layer by layer."""
        T = tokens.total_length
        arr = lambda x: tokens._with_values(x)  # noqa: E731  (same sequences, other values)
        x = self.embed[tokens.values]
        for i, lay in enumerate(self.layers):
            qkv = rmsnorm_qkv(x, None, lay["qkv"]).view(T, HEADS + 2 * KV_HEADS, DIM)
            q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], dim=1)  # strided views, no copies
            paged.paged_write(cache, i, slots, arr(k), arr(v))
            a = paged.paged_attention(arr(q), cache, i, slots, mask=mask).values
            x = x + a.reshape(T, -1) @ lay["out"]
            x = x + torch.relu(varlen_rmsnorm_triton(x) @ lay["up"]) @ lay["down"]
        return varlen_rmsnorm_triton(x) @ self.head


def packed(rows, device):
    """An Array of int64 ids from lists."""
    host = [0]
    for r in rows:
        host.append(host[-1] + len(r))
    vals = torch.tensor([t for r in rows for t in r], dtype=torch.int64, device=device)
    return scree.Array(vals, torch.tensor(host, dtype=torch.int32, device=device), _host=tuple(host))


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def step(model, cache, slots, trees, parents):
    """Reserves room for the trees, runs the model over them; logits and the grown cache."""
    dev = slots.device
    tokens = packed(trees, dev)
    cache = paged.paged_reserve(cache, slots, i32([len(t) for t in trees], dev))
    mask = None
    if parents is not None:
        mask = paged.tree_mask(tokens._with_values(i32([p for row in parents for p in row], dev)))
    return model(tokens, cache, slots, mask), cache


def greedy(model, prompts, new_tokens, device):
    """One token a step."""
    cache, slots = new_cache(prompts, new_tokens, device)
    logits, cache = step(model, cache, slots, prompts, None)
    ends = torch.tensor([len(p) for p in prompts]).cumsum(0) - 1
    last = logits[ends.to(device)].argmax(-1).tolist()
    out = [[t] for t in last]
    for _ in range(new_tokens - 1):
        logits, cache = step(model, cache, slots, [[o[-1]] for o in out], None)
        for b, t in enumerate(logits.argmax(-1).tolist()):
            out[b].append(t)
    return out


def draft(logits_row, first, truth, rng):
    """A tree under token `first`: two guesses a level, the likeliest alternatives of the last
    logits; `truth` (what a good draft model would say) is mixed in to have something to accept."""
    alts = logits_row.topk(4).indices.tolist()
    tokens, parents = [first], [-1]
    frontier = [0]
    for depth in range(3):
        nxt = []
        for node in frontier[:2]:
            for guess in (alts[int(torch.randint(4, (1,), generator=rng))],
                          truth[depth] if depth < len(truth) and torch.rand(1, generator=rng) < 0.7 else alts[0]):
                tokens.append(guess)
                parents.append(node)
                nxt.append(len(tokens) - 1)
        frontier = nxt[::-1]
    return tokens, parents


def new_cache(prompts, new_tokens, device):
    B = len(prompts)
    width = (max(map(len, prompts)) + new_tokens + 40) // PAGE + 2
    cache = paged.paged_cache(LAYERS, B * width, PAGE, KV_HEADS, DIM, B, width, device=device)
    return cache, torch.arange(B, dtype=torch.int32, device=device)


def speculative(model, prompts, new_tokens, device, truth, seed=1):
    """Greedy decoding, a drafted tree a step; tokens, model steps, and their log probabilities."""
    rng = torch.Generator().manual_seed(seed)
    B = len(prompts)
    cache, slots = new_cache(prompts, new_tokens, device)
    logits, cache = step(model, cache, slots, prompts, None)
    ends = torch.tensor([len(p) for p in prompts]).cumsum(0) - 1
    rows = logits[ends.to(device)]
    out, logps, steps = [[] for _ in range(B)], [[] for _ in range(B)], 0
    pending = rows.argmax(-1).tolist()  # each sequence's next token, known but not yet cached
    while min(map(len, out)) < new_tokens:
        trees, parents = zip(*(draft(rows[b], pending[b], truth[b][len(out[b]) + 1:], rng) for b in range(B)))
        logits, cache = step(model, cache, slots, trees, parents)
        steps += 1
        picks, paths, rows, at = logits.argmax(-1).tolist(), [], [], 0
        for b in range(B):
            node, path = 0, [0]
            while True:  # follow the child that greedy decoding would have produced
                want = picks[at + node]
                child = [c for c in range(len(trees[b])) if parents[b][c] == node and trees[b][c] == want]
                if not child:
                    break
                node = child[0]
                path.append(node)
            out[b] += [trees[b][i] for i in path]
            paths.append(path)
            rows.append(at + node)
            pending[b] = picks[at + node]
            at += len(trees[b])
        # Scores of the tokens that follow the accepted ones, with two alternatives each.
        said = torch.full((at,), -100, dtype=torch.int64, device=device)
        said[torch.tensor(rows, device=device)] = torch.tensor(pending, device=device)
        scores = token_logprobs(logits, said, top_k=2)
        for b, lp in enumerate(scores.logp[torch.tensor(rows, device=device)].tolist()):
            logps[b].append(lp)
        rows = logits[torch.tensor(rows, device=device)]
        depth = max(map(len, paths))
        cache = paged.paged_accept(cache, slots, i32([len(t) for t in trees], device),
                                   i32([p + [-1] * (depth - len(p)) for p in paths], device))
    _lib.raise_device_status()
    return [o[:new_tokens] for o in out], steps, logps, cache


def main(device="cuda:0", new_tokens=24):
    device = torch.device(device)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(VOCAB, (n,), generator=g).tolist() for n in (5, 40, 17, 128)]
    model = Decoder(device)
    plain = greedy(model, prompts, new_tokens, device)
    spec, steps, logps, cache = speculative(model, prompts, new_tokens, device, plain)
    same = sum(a == b for p, s in zip(plain, spec) for a, b in zip(p, s))
    # Two samples that go on from the first sequence's prefix, which they share; the other
    # sequences end, and the pages in use move to the front of the pools.
    slots = torch.arange(len(prompts), dtype=torch.int32, device=device)
    cache = paged.paged_free(cache, slots[1:])
    cache = paged.paged_fork(cache, slots[:1].repeat(2), slots[1:3])
    cache = paged.paged_compact(cache)
    _lib.raise_device_status()
    print(f"{len(prompts)} sequences, {new_tokens} tokens each in {steps} steps of the model "
          f"({same} of {new_tokens * len(prompts)} tokens as in plain decoding); "
          f"mean log probability {sum(map(sum, logps)) / sum(map(len, logps)):.2f}; "
          f"{int((cache.refs > 0).sum())} pages in use after two forks")
    return plain, spec, steps, cache


if __name__ == "__main__":
    main()
