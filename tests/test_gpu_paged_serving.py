"""PagedCache and the example that uses it: the bookkeeping of pages over many steps, against the definition in 64 bits."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _cache(**kw):
    import shmtensor_amd
    shmtensor_amd.install_aliases()
    from shmtensor_amd.shmtensor import PagedCache
    return PagedCache(**kw)


def _attended(cache, step, layer, q, got, **kw):
    """Against the definition: one rounding of the result to bfloat16, one of each weight (2^-9 each), twice."""
    out, _, spread, _ = paged.attention(q.double().cpu().numpy(), cache.cache[layer].cpu().numpy(),
                                        cache.scales[layer].cpu().numpy(), cache.block_table.cpu().numpy(),
                                        step.query_starts.cpu().numpy(), step.kv_lens.cpu().numpy(), q.shape[2] ** -0.5, **kw)
    far = np.abs(got.double().cpu().numpy() - out)
    assert (far <= 2.0 ** -8 * (np.abs(out) + spread) + 1e-4 * spread + 1e-30).all(), far.max()


@pytest.mark.parametrize("window, sinks", [(0, 0), (24, 5)])
def test_steps_of_many_requests(window, sinks):
    gen = torch.Generator().manual_seed(2)
    rng = np.random.default_rng(2)
    cache = _cache(pages=40, kv_heads=2, dim=64, requests=5, max_len=200, layers=2)
    held = {}                                                          # request -> the rows that it was given, as stored
    for turn in range(30):
        new = rng.integers(0, 9, 5) * (rng.random(5) < 0.7)
        for r in range(5):
            if cache.lens[r] > 150 or rng.random() < 0.03:
                cache.release(r)
                held.pop(r, None)
        before = cache.lens.copy()
        step = cache.plan(new)
        assert step.tokens == new.sum() and step.kv_lens.tolist() == (before + new).tolist()
        n = step.tokens
        q, k, v = (torch.randn((n, h, 64), generator=gen).bfloat16().cuda() for h in (6, 2, 2))
        for layer in range(2):
            cache.set(step, layer, k, v * (layer + 1))
            got = cache.attend(step, layer, q, window=window, sinks=sinks)
            _attended(cache, step, layer, q, got, window=window, sinks=sinks)
        code, byte = paged.encode(k.double().cpu().numpy())
        assert np.array_equal(cache.fetch(step, 1, torch.float32)[0].double().cpu().numpy(), paged.decode(code, byte))
        at = 0
        for r in range(5):
            held.setdefault(r, []).append(k[at:at + new[r]])
            at += new[r]
        used = cache.block_table[cache.block_table >= 0].tolist() + cache._free.tolist()
        assert sorted(used) == list(range(40)), "a page is lost or has two owners"
        if window:
            for r in range(5):
                cache.trim(r, window, sinks)
    assert window == 0 or int((cache.block_table >= 0).sum()) <= 5 * 5


def test_refusals_change_nothing():
    cache = _cache(pages=4, kv_heads=1, dim=64, requests=2, max_len=60)
    cache.plan([17, 0])
    for bad, text in (([30, 20], "pages needed"), ([50, 0], "beyond max_len"), ([1], "for each"), ([-1, 0], "for each")):
        with pytest.raises((RuntimeError, ValueError), match=text):
            cache.plan(bad)
    assert cache.free_pages == 2 and cache.lens.tolist() == [17, 0]
    step = cache.plan([15, 32])
    assert cache.free_pages == 0 and sorted(cache.block_table[cache.block_table >= 0].tolist()) == [0, 1, 2, 3]
    assert step.kv_lens.tolist() == [32, 32]


def test_the_example_runs_and_repeats_itself():
    """Two runs give the same tokens: nothing in the operators depends on an order that may change."""
    spec = importlib.util.spec_from_file_location("paged_generation", os.path.join(ROOT, "examples", "paged_generation.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 1024, (n,), generator=gen).tolist() for n in (5, 90, 33)]
    for window, sinks in ((0, 0), (48, 4)):
        answers = example.generate(prompts, 12, window, sinks)
        assert [len(a) for a in answers] == [12] * 3 and all(0 <= t < 1024 for a in answers for t in a)
        assert answers == example.generate(prompts, 12, window, sinks)
