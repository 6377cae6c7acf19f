"""PagedCache over steps of drafted trees, in 4 and 8 bits, and over an encoder's states: plan, rows, attention, kept paths,
pages that come back, against the definition in 64 bits; and the example that uses them."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from oracle import paged_more
from test_gpu_paged_tree import grown

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"


def _cache(**kw):
    import shmtensor_amd
    shmtensor_amd.install_aliases()
    from shmtensor_amd.shmtensor import PagedCache
    return PagedCache(**kw)


def _np(t):
    return (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t).cpu().numpy()


def _attended(cache, layer, q, got, starts, kv_lens, **kw):
    """As in test_gpu_paged_serving.py: one rounding of the result to bfloat16, one of each weight (2^-9 each), twice."""
    out, _, spread, _ = paged_more.attention(q.double().cpu().numpy(), _np(cache.cache[layer]), _np(cache.scales[layer]),
                                             _np(cache.block_table), starts, kv_lens, q.shape[2] ** -0.5, cache.bits, **kw)
    far = np.abs(got.double().cpu().numpy() - out)
    assert (far <= 2.0 ** -8 * (np.abs(out) + spread) + 1e-4 * spread + 1e-30).all(), far.max()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("window, sinks", [(0, 0), (24, 5)])
def test_steps_of_trees_and_chains(bits, window, sinks):
    gen = torch.Generator().manual_seed(bits)
    rng = np.random.default_rng(bits)
    cache = _cache(pages=60, kv_heads=2, dim=64, requests=5, max_len=200, layers=2, bits=bits)
    want_rows = [np.zeros((2, 0, 2, 64)) for _ in range(5)]            # what each request's tokens were given, layer 0: keys, values
    lens = np.zeros(5, np.int64)
    for turn in range(30):
        for r in range(5):
            if lens[r] > 150 or rng.random() < 0.05:
                cache.release(r)
                lens[r], want_rows[r] = 0, np.zeros((2, 0, 2, 64))
        new = rng.integers(0, 14, 5) * (rng.random(5) < 0.8)
        as_trees = turn % 3 > 0
        parents = np.concatenate([grown(rng, n, ("tree", "late", "forest")[r % 3]) for r, n in enumerate(new)]).astype(np.int64)
        step = cache.plan(new, parents=parents if turn % 2 else torch.from_numpy(parents).int().to(DEV)) if as_trees else cache.plan(new)
        n, starts, total = step.tokens, np.concatenate([[0], np.cumsum(new)]), lens + new
        assert n == new.sum() and step.kv_lens.tolist() == total.tolist()
        if as_trees:
            nodes, positions = paged_more.tree(parents, starts, total)
            assert np.array_equal(_np(step.nodes), nodes) and np.array_equal(_np(step.positions), positions)
        q, k, v = (torch.randn((n, h, 64), generator=gen).bfloat16().to(DEV) for h in (6, 2, 2))
        for layer in range(2):
            cache.set(step, layer, k, v * (layer + 1))
            got = cache.attend(step, layer, q, window=window, sinks=sinks)
            _attended(cache, layer, q, got, starts, total, window=window, sinks=sinks,
                      **(dict(seen="tree", parents=parents) if as_trees else {}))
        rows = np.stack([k.double().cpu().numpy(), v.double().cpu().numpy()])
        for r in range(5):
            want_rows[r] = np.concatenate([want_rows[r], rows[:, starts[r]:starts[r + 1]]], 1)
        if as_trees:
            tokens, picked = rng.integers(0, 3, n), rng.integers(0, 3, n)
            if window:
                cache.trim(int(rng.integers(5)), window, sinks)        # before it is known what stays: what could be seen stays
            there = [torch.from_numpy(x).to(DEV) for x in (tokens, picked)]
            empty = np.zeros((1, 0, 2, 2, 16, 32 * bits // 4), np.uint8), np.zeros((1, 0, 2, 2, 2, 16), np.uint8)
            counts, path, after = paged_more.keep(*empty, _np(cache.block_table), starts, total, parents, tokens, picked)
            got_counts, got_path, got_after = cache.keep(step, *there)
            assert got_counts.tolist() == counts.tolist() and got_path.tolist() == path.tolist()
            assert got_after.tolist() == after.tolist()
            for r in range(5):
                kept = path[starts[r]:starts[r] + counts[r]]
                want_rows[r] = want_rows[r][:, list(range(lens[r])) + [lens[r] + int(x) for x in kept]]
            total = lens + counts
        lens = total
        assert cache.lens.tolist() == lens.tolist() and cache._kv_lens.tolist() == lens.tolist()
        used = cache.block_table[cache.block_table >= 0].tolist() + cache._free.tolist()
        assert sorted(used) == list(range(60)), "a page is lost or has two owners"
        if window:
            for r in range(5):
                cache.trim(r, window, sinks)
        encode = paged_more.encode8 if bits == 8 else paged_more.paged.encode
        decode = paged_more.decode8 if bits == 8 else paged_more.paged.decode
        for r in range(5):                                             # what is still there is what was given, rounded once
            table = _np(cache.block_table)[r]
            j = np.array([x for x in range(lens[r]) if table[x // 16] >= 0], int)
            if len(j) == 0:
                continue
            held = paged_more.rows_fetch(_np(cache.cache[0]), _np(cache.scales[0]), table[j // 16] * 16 + j % 16, bits)
            for have, given in zip(held, want_rows[r]):
                assert np.array_equal(have, decode(*encode(given[j])))


def test_an_encoders_states():
    gen = torch.Generator().manual_seed(1)
    for bits in (4, 8):
        states = _cache(pages=30, kv_heads=3, dim=128, requests=3, max_len=200, page=32, bits=bits)
        step = states.plan([70, 0, 190])
        k, v = (torch.randn((260, 3, 128), generator=gen).half().to(DEV) for _ in range(2))
        states.set(step, 0, k, v)
        for news in ([5, 2, 5], [1, 0, 90]):
            q = torch.randn((sum(news), 6, 128), generator=gen).half().to(DEV)
            starts = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device=DEV)
            got, lse = states.attend_all(0, q, starts, max_query_len=max(news), return_lse=True)
            _attended(states, 0, q, got, _np(starts), np.array([70, 0, 190]), seen="all")
            assert bool((got[news[0]:news[0] + news[1]] == 0).all()) and bool(lse[news[0]:news[0] + news[1]].isneginf().all())


def test_refusals_change_nothing():
    cache = _cache(pages=4, kv_heads=1, dim=64, requests=2, max_len=60)
    with pytest.raises(ValueError, match="4 or 8 bits"):
        _cache(pages=4, kv_heads=1, dim=64, requests=2, max_len=60, bits=6)
    with pytest.raises(ValueError, match="each of 5 new tokens"):
        cache.plan([3, 2], parents=[-1, 0])
    assert cache.lens.tolist() == [0, 0] and cache.free_pages == 4
    plain = cache.plan([3, 2])
    ints = torch.zeros(5, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="no trees"):
        cache.keep(plain, ints, ints)
    step = cache.plan([3, 2], parents=[-1, 0, 0, -1, 0])
    cache.plan([1, 1])
    with pytest.raises(ValueError, match="not the last one"):
        cache.keep(step, ints, ints)
    step = cache.plan([3, 2], parents=[-1, 0, 0, -1, 0])
    with pytest.raises(RuntimeError, match="each of 5 nodes"):
        cache.keep(step, ints[:4], ints[:4])
    assert cache.lens.tolist() == [10, 7]
    counts, _, _ = cache.keep(step, ints, ints)
    with pytest.raises(ValueError, match="not the last one"):
        cache.keep(step, ints, ints)
    assert counts.tolist() == [2, 2] and cache.lens.tolist() == [9, 7]


def test_the_example_runs_with_drafts():
    spec = importlib.util.spec_from_file_location("paged_generation", os.path.join(ROOT, "examples", "paged_generation.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.draft([5, 1, 2, 5, 1, 3, 5], 2, 2) == ([5, 1, 3, 2], [-1, 0, 1, 1])
    gen = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 40, (n,), generator=gen).tolist() for n in (5, 90, 33)]
    for bits, window, sinks in ((4, 0, 0), (8, 48, 4)):
        answers, taken = example.generate_drafted(prompts, 12, 3, window=window, sinks=sinks, bits=bits)
        assert all(len(a) >= 12 for a in answers) and taken <= 12 and all(0 <= t < 1024 for a in answers for t in a)
        assert (answers, taken) == example.generate_drafted(prompts, 12, 3, window=window, sinks=sinks, bits=bits)
        plain = example.generate(prompts, 12, window, sinks, bits=bits)
        assert [len(a) for a in plain] == [12] * 3
