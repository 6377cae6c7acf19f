"""Drafted steps from end to end: what is kept is what the model says, in fewer steps than tokens; steps whose first nodes are text
(a prompt with a tree behind it); requests that are released while their step runs. Against definitions and known answers."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from oracle import paged_more
from test_gpu_paged_drafting import _cache, _np
from test_gpu_paged_keep import Step
from test_gpu_paged_tree import _check, grown

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"


@pytest.fixture
def example():
    spec = importlib.util.spec_from_file_location("paged_generation", os.path.join(ROOT, "examples", "paged_generation.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


class Cycle:
    """A model whose answer is known: behind token t comes t + 1, behind the last of `period` the first. The attention runs, over
    rows that say nothing about the answer, and its result is multiplied by 0."""

    def __init__(self, decoder, period):
        self.layers, self.heads, self.kv_heads, self.dim = decoder.layers, decoder.heads, decoder.kv_heads, decoder.dim
        self.decoder, self.period = decoder, period

    def logits(self, tokens, step, cache, window, sinks, every=False):
        idle = self.decoder.logits(tokens, step, cache, window, sinks, every=True)
        said = torch.nn.functional.one_hot((tokens + 1) % self.period, idle.shape[1]) + 0 * idle.float()
        return said if every else said[step.query_starts[1:].long() - 1]


@pytest.mark.parametrize("bits, window, sinks", [(4, 0, 0), (8, 48, 4)])
def test_drafts_that_are_right_save_steps(example, bits, window, sinks):
    """Prompts that hold the cycle more than once: every draft of 3 tokens is right, so a step brings 4. From the prompts' step on,
    which brings one, 13 tokens take 1 + 3 steps, and the answers are the cycle's."""
    model = Cycle(example.Decoder(), 7)
    prompts = [[t % 7 for t in range(n)] for n in (20, 90, 33)]
    answers, taken = example.generate_drafted(prompts, 13, 3, window=window, sinks=sinks, model=model, bits=bits)
    assert answers == [[t % 7 for t in range(len(p), len(p) + 13)] for p in prompts]
    assert taken == 4
    assert example.generate(prompts, 13, window, sinks, model=model, bits=bits) == answers


def test_drafts_that_are_wrong_cost_only_themselves(example):
    """Prompts in which the tokens behind are drawn: few drafts are right. Answers and steps as a walk down the trees has them."""
    model = Cycle(example.Decoder(), 11)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 11, n).tolist() for n in (60, 25)]
    texts, steps = [p + [(p[-1] + 1) % 11] for p in prompts], 1
    while min(len(t) - len(p) for t, p in zip(texts, prompts)) < 9:
        for t, p in zip(texts, prompts):
            if len(t) - len(p) >= 9:
                continue
            nodes, parents = example.draft(t, 3, 2)
            at = 0
            while at is not None:
                t.append((nodes[at] + 1) % 11)
                at = next((c for c in range(len(nodes)) if parents[c] == at and nodes[c] == t[-1]), None)
        steps += 1
    answers, taken = example.generate_drafted(prompts, 9, 3, model=model)
    assert answers == [t[len(p):] for t, p in zip(texts, prompts)] and taken == steps
    assert all(a == [(p[-1] + 1 + i) % 11 for i in range(len(a))] for p, a in zip(prompts, answers))


def _prompt_with_tree(rng, text, drafts):
    """Parents of `text` nodes in a row, and a tree below the last of them."""
    tree = grown(rng, drafts + 1, "tree")                               # its root is the text's last node
    return np.concatenate([np.arange(text) - 1, tree[1:] + text - 1])


@pytest.mark.parametrize("text", [1, 40, 63, 64, 65, 500, 1000, 1015, 1024, 3000])
@pytest.mark.parametrize("drafts", [1, 2, 20, 64])
def test_trees_behind_a_prompt_are_numbered(capi, text, drafts):
    rng = np.random.default_rng(text + drafts)
    parents = [_prompt_with_tree(rng, n, drafts) for n in (text, 7)]
    starts = np.cumsum([0] + [len(p) for p in parents])
    _check(capi, np.concatenate(parents), starts, [text + drafts + 100, drafts + 7])


@pytest.mark.parametrize("bits", [4, 8])
def test_trees_behind_a_prompt_are_kept(capi, bits):
    news, given = [520, 1090, 30, 64, 5], [500, 1026, 1, 64, 3]
    s = Step(bits, [0, 70, 9, 3, 16], news, bits=bits, heads=2)
    for b, (n, g) in enumerate(zip(news, given)):
        lo = int(s.starts[b])
        s.parents[lo:lo + n] = _prompt_with_tree(s.rng, g, n - g)
        for i in range(g - 1, n):                                       # from the text's end on somebody follows, mostly
            kids = [c for c in range(i + 1, n) if s.parents[lo + c] == i]
            if kids and s.rng.random() < 0.9:
                s.picked[lo + i] = s.tokens[lo + kids[-1]]
    counts = s.check(capi, given=given)
    assert (counts.cpu().numpy() >= given).all() and int((counts.cpu().numpy() - given).max()) >= 2


@pytest.mark.parametrize("bits", [4, 8])
def test_a_request_is_released_while_its_step_runs(bits):
    """The others' paths and rows are the definition's, the released one's pages are untouched until somebody else has them."""
    rng = np.random.default_rng(bits)
    cache = _cache(pages=30, kv_heads=2, dim=64, requests=3, max_len=150, layers=2, bits=bits)
    new = np.array([50, 37, 90])
    rows = lambda n: [torch.from_numpy(rng.standard_normal((n, 2, 64))).bfloat16().to(DEV) for _ in range(2)]
    step = cache.plan(new)
    for layer in range(2):
        cache.set(step, layer, *rows(step.tokens))
    drafts = np.array([12, 9, 20])
    parents = np.concatenate([grown(rng, n, "late") for n in drafts])
    step = cache.plan(drafts, parents=parents)
    for layer in range(2):
        cache.set(step, layer, *rows(step.tokens))
    cache.release(1)
    tokens, picked = rng.integers(0, 2, 41), rng.integers(0, 2, 41)
    held = _np(cache.cache).copy(), _np(cache.scales).copy()
    starts = np.concatenate([[0], np.cumsum(drafts)])
    counts, path, after = paged_more.keep(*held, _np(cache.block_table), starts, new + drafts, parents, tokens, picked)
    counts[1], path[12:21], after[1] = 0, -1, -1
    got = cache.keep(step, torch.from_numpy(tokens).to(DEV), torch.from_numpy(picked).to(DEV))
    assert got[0].tolist() == counts.tolist() and got[1].tolist() == path.tolist() and got[2].tolist() == after.tolist()
    assert np.array_equal(_np(cache.cache), held[0]) and np.array_equal(_np(cache.scales), held[1])
    lens = np.array([50, 0, 90]) + counts
    assert cache.lens.tolist() == lens.tolist() == cache._kv_lens.tolist()
    used = cache.block_table[cache.block_table >= 0].tolist() + cache._free.tolist()
    assert sorted(used) == list(range(30)) and (cache.block_table[1] < 0).all()
    step = cache.plan([1, 40, 1])
    assert step.kv_lens.tolist() == (lens + [1, 40, 1]).tolist() and (step.slots >= 0).all()
