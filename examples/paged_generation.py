"""A small decoder with random weights answers a batch of prompts from a paged cache held in 4 bits: prompts at once, then a
token a step, requests of different lengths side by side, with a window and a few first tokens that stay visible.

    python examples/paged_generation.py --steps 64 --window 256 --sinks 4
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

    def logits(self, tokens, step, cache, window, sinks):
        """Logits of each request's last token in this step."""
        x = self.embed[tokens]
        turn = step.positions.float()[:, None] * torch.exp2(-torch.arange(x.shape[1], device=x.device) / 32.0)
        x = x + torch.cos(turn).bfloat16() @ self.place
        for layer in range(self.layers):
            y = (x @ self.qkv[layer]).view(len(x), self.heads + 2 * self.kv_heads, self.dim)
            q, k, v = y.split([self.heads, self.kv_heads, self.kv_heads], 1)
            cache.set(step, layer, k, v)
            a = cache.attend(step, layer, q, window=window, sinks=sinks)
            x = x + a.flatten(1) @ self.out[layer]
        last = step.query_starts[1:].long() - 1
        return x[last] @ self.head


def generate(prompts, steps, window=0, sinks=0, model=None, page=16):
    """Greedy continuations of the prompts (lists of token ids): a list of lists."""
    model = model or Decoder()
    longest = max(len(p) for p in prompts) + steps
    pages = sum(-(-(len(p) + steps) // page) for p in prompts)
    cache = PagedCache(pages, model.kv_heads, model.dim, len(prompts), longest, layers=model.layers, page=page)
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


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=4)
    args = ap.parse_args()
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1024, (50 + 37 * r,), generator=gen).tolist() for r in range(args.requests)]
    generate(prompts, 2, args.window, args.sinks)
    torch.cuda.synchronize()
    t = time.perf_counter()
    answers = generate(prompts, args.steps, args.window, args.sinks)
    t = time.perf_counter() - t
    print("first answer:", answers[0][:16], "...")
    print("%d requests, %d tokens each: %.0f tokens/s" % (len(prompts), args.steps, len(prompts) * args.steps / t))
