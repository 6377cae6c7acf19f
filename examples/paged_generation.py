"""A small decoder with random weights answers a batch of prompts from a paged cache held in 4 or 8 bits: prompts at once, then a
token a step, requests of different lengths side by side, with a window and a few first tokens that stay visible. With --drafts
a step takes what followed the last token's earlier occurrences as a tree of drafted tokens, and keeps the path that the model
agrees with.

    python examples/paged_generation.py --steps 64 --window 256 --sinks 4
    python examples/paged_generation.py --steps 64 --bits 8 --drafts 3
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from shmtensor_amd.shmtensor import PagedCache  # noqa: E402


class Decoder:
    def __init__(self, vocab=1024, layers=2, heads=8, kv_heads=2, dim=64, device="cuda", seed=0):
        gen = torch.Generator(device=device).manual_seed(seed)
        width = heads * dim
        def w(*shape):
            return torch.randn(shape, generator=gen, device=device, dtype=torch.float32).mul_(shape[0] ** -0.5).bfloat16()
        self.heads, self.kv_heads, self.dim, self.layers = heads, kv_heads, dim, layers
        self.embed = torch.randn((vocab, width), generator=gen, device=device).bfloat16()
        self.place = w(width, width)
        self.qkv = [w(width, (heads + 2 * kv_heads) * dim) for _ in range(layers)]
        self.out = [w(width, width) for _ in range(layers)]
        self.head = w(width, vocab)

    def logits(self, tokens, step, cache, window, sinks, every=False):
        """Logits of each request's last token in this step, or of every token."""
        x = self.embed[tokens]
        turn = step.positions.float()[:, None] * torch.exp2(-torch.arange(x.shape[1], device=x.device) / 32.0)
        x = x + torch.cos(turn).bfloat16() @ self.place
        for layer in range(self.layers):
            y = (x @ self.qkv[layer]).view(len(x), self.heads + 2 * self.kv_heads, self.dim)
            q, k, v = y.split([self.heads, self.kv_heads, self.kv_heads], 1)
            cache.set(step, layer, k, v)
            a = cache.attend(step, layer, q, window=window, sinks=sinks)
            x = x + a.flatten(1) @ self.out[layer]
        if every:
            return x @ self.head
        last = step.query_starts[1:].long() - 1
        return x[last] @ self.head


def generate(prompts, steps, window=0, sinks=0, model=None, page=16, bits=4):
    """Greedy continuations of the prompts (lists of token ids): a list of lists."""
    model = model or Decoder()
    longest = max(len(p) for p in prompts) + steps
    pages = sum(-(-(len(p) + steps) // page) for p in prompts)
    cache = PagedCache(pages, model.kv_heads, model.dim, len(prompts), longest, layers=model.layers, page=page, bits=bits)
    tokens = torch.tensor([t for p in prompts for t in p], device="cuda")
    new = [len(p) for p in prompts]
    answers = []
    for _ in range(steps):
        step = cache.plan(new)
        tokens = model.logits(tokens, step, cache, window, sinks).argmax(-1)
        answers.append(tokens)
        new = [1] * len(prompts)
        if window:
            for r in range(len(prompts)):
                cache.trim(r, window, sinks)
    return torch.stack(answers, 1).tolist()


def draft(text, depth, branches):
    """A tree of what may follow: the last token, and below it what came after its latest earlier occurrences. (tokens, parents)"""
    tokens, parents = [text[-1]], [-1]
    found = [i for i in range(len(text) - 2, -1, -1) if text[i] == text[-1]][:branches]
    for i in found:
        at = 0
        for t in text[i + 1:min(i + 1 + depth, len(text))]:
            twin = [c for c in range(1, len(tokens)) if parents[c] == at and tokens[c] == t]
            if not twin:
                tokens.append(t)
                parents.append(at)
            at = twin[0] if twin else len(tokens) - 1
    return tokens, parents


def generate_drafted(prompts, steps, depth, branches=2, window=0, sinks=0, model=None, page=16, bits=4):
    """Continuations of `steps` tokens and more, a path of a tree a step: (list of lists, steps that it took)."""
    model = model or Decoder()
    most = 1 + depth * branches
    longest = max(len(p) for p in prompts) + steps + 2 * most
    pages = sum(-(-(len(p) + steps + 2 * most) // page) for p in prompts)
    cache = PagedCache(pages, model.kv_heads, model.dim, len(prompts), longest, layers=model.layers, page=page, bits=bits)
    tokens = torch.tensor([t for p in prompts for t in p], device="cuda")
    step = cache.plan([len(p) for p in prompts])
    following = model.logits(tokens, step, cache, window, sinks).argmax(-1).tolist()
    texts = [list(p) + [t] for p, t in zip(prompts, following)]
    taken = 1
    while min(len(t) - len(p) for t, p in zip(texts, prompts)) < steps:
        # a request that has its tokens waits for the others
        trees = [draft(t, depth, branches) if len(t) - len(p) < steps else ([], []) for t, p in zip(texts, prompts)]
        tokens = torch.tensor([t for tree in trees for t in tree[0]], device="cuda")
        step = cache.plan([len(tree[0]) for tree in trees], parents=[p for tree in trees for p in tree[1]])
        picked = model.logits(tokens, step, cache, window, sinks, every=True).argmax(-1)
        counts, path, token = cache.keep(step, tokens, picked)
        path, token, at = path.tolist(), token.tolist(), 0
        for r, (tree, _) in enumerate(trees):
            if tree:
                texts[r] += [tree[path[at + k]] for k in range(1, counts[r])] + [token[r]]
            at += len(tree)
        taken += 1
        if window:
            for r in range(len(prompts)):
                cache.trim(r, window, sinks)
    return [t[len(p):] for t, p in zip(texts, prompts)], taken


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=4)
    ap.add_argument("--bits", type=int, default=4, choices=(4, 8))
    ap.add_argument("--drafts", type=int, default=0, help="drafted tokens in a row; 0: none")
    args = ap.parse_args()
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1024, (50 + 37 * r,), generator=gen).tolist() for r in range(args.requests)]
    def run(steps):
        if args.drafts:
            return generate_drafted(prompts, steps, args.drafts, window=args.window, sinks=args.sinks, bits=args.bits)
        return generate(prompts, steps, args.window, args.sinks, bits=args.bits), steps
    run(2)
    torch.cuda.synchronize()
    t = time.perf_counter()
    answers, taken = run(args.steps)
    t = time.perf_counter() - t
    print("first answer:", answers[0][:16], "...")
    print("%d requests, %d tokens each in %d steps: %.0f tokens/s" % (len(prompts), args.steps, taken, sum(map(len, answers)) / t))
