"""The accepted path of a tree of drafted tokens and its rows (page_keep): bit for bit the definition (oracle/paged_more.py)."""
import numpy as np
import pytest
import torch

from oracle import paged_more
from test_gpu_paged_tree import grown

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Step:
    """Requests with pages of random bytes, in which a few of a node's children have the token that was picked."""

    def __init__(self, seed, cached, news, bits=4, heads=2, dim=64, page=16, layers=2, agree=0.9, kinds=("tree", "late", "chain", "forest")):
        rng = self.rng = np.random.default_rng(seed)
        news, cached = np.asarray(news), np.asarray(cached)
        total = cached + news
        width = max(1, int((-(-total // page)).max(initial=0)))
        count = -(-total // page)
        pages = int(count.sum()) + 2
        order = rng.permutation(pages)
        self.table = np.full((len(news), width), -1, np.int32)
        at = 0
        for b, c in enumerate(count):
            self.table[b, :c] = order[at:at + c]
            at += c
        self.cache = rng.integers(0, 256, (layers, pages, heads, 2, page, dim * bits // 8), np.uint8)
        self.scales = rng.integers(0, 256, (layers, pages, heads, 2, dim // 32, page), np.uint8)
        self.starts, self.lens, self.bits = np.concatenate([[0], np.cumsum(news)]), total, bits
        n = int(self.starts[-1])
        self.parents = np.concatenate([grown(rng, k, kinds[i % len(kinds)]) for i, k in enumerate(news)] + [np.zeros(0, int)])
        self.tokens, self.picked = rng.integers(0, 9, n), rng.integers(0, 9, n)
        for b, k in enumerate(news):                                    # mostly, somebody follows
            lo = int(self.starts[b])
            for i in range(k):
                kids = [c for c in range(k) if self.parents[lo + c] == i]
                if kids and rng.random() < agree:
                    self.picked[lo + i] = self.tokens[lo + kids[int(rng.integers(len(kids)))]]

    def check(self, capi, dtype=torch.int64, len_dtype=torch.int32, given=None, whole=True):
        put = lambda x, t: torch.tensor(np.asarray(x), dtype=t, device=DEV)
        cache, scales = put(self.cache, torch.uint8), put(self.scales, torch.uint8)
        there = cache.view(torch.float8_e4m3fn) if self.bits == 8 else cache
        args = there, scales
        if not whole:
            args = there[0], scales[0]
        counts, path, after = capi.page_keep(*args, put(self.table, torch.int32), put(self.starts, len_dtype),
                                             put(self.lens, len_dtype), put(self.parents, torch.int32), put(self.tokens, dtype),
                                             put(self.picked, dtype), None if given is None else put(given, torch.int32))
        held = (self.cache.copy(), self.scales.copy()) if whole else (self.cache[:1].copy(), self.scales[:1].copy())
        want = paged_more.keep(*held, self.table, self.starts, self.lens, self.parents, self.tokens, self.picked, given)
        assert counts.dtype == path.dtype == torch.int32 and after.dtype == dtype
        for g, w in zip((counts, path, after), want):
            assert np.array_equal(g.cpu().numpy(), w)
        k = self.cache.shape[0] if whole else 1
        assert np.array_equal(cache[:k].cpu().numpy(), held[0]) and np.array_equal(scales[:k].cpu().numpy(), held[1])
        assert np.array_equal(cache[k:].cpu().numpy(), self.cache[k:])
        return counts


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_paths_and_rows(capi, bits, dim, page):
    s = Step(dim + page, [0, 5, 31, 100, 16, 3, 250], [1, 7, 33, 64, 0, 20, 11], bits=bits, dim=dim, page=page, heads=3)
    assert int(s.check(capi).max()) >= 2                               # somebody follows


@pytest.mark.parametrize("layers, heads", [(1, 1), (1, 5), (7, 3), (24, 8)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_layers_and_heads(capi, layers, heads, dtype):
    Step(layers, [40, 9], [30, 64], layers=layers, heads=heads).check(capi, dtype, dtype)


def test_long_paths(capi):
    """More moves than one round of the list, nodes beyond the first 64, rows of a place read before it is written."""
    s = Step(3, [20, 0, 7], [900, 300, 70], kinds=("late",), agree=1.0, dim=64, heads=1)
    assert int(s.check(capi).max()) > 20
    s = Step(4, [2], [700], kinds=("chain",), heads=1)
    s.parents[1:] = np.arange(699)
    s.parents[1], s.parents[2] = 0, 0                                   # everything is one place too far
    s.tokens[:], s.picked[:] = 1, 1
    s.tokens[1] = 2
    assert s.check(capi).tolist() == [699]


def test_many_requests(capi):
    rng = np.random.default_rng(5)
    Step(5, rng.integers(0, 60, 150), rng.integers(0, 40, 150), heads=1).check(capi)
    Step(6, rng.integers(0, 9, 3000), rng.integers(0, 4, 3000), heads=1, layers=1).check(capi)


def test_given_tokens(capi):
    s = Step(7, [10, 0, 33, 5, 8], [12, 90, 64, 0, 9], kinds=("late",))
    for b, g in enumerate([12, 60, 1, 0, 4]):
        lo = int(s.starts[b])
        s.parents[lo:lo + g] = np.arange(g) - 1
    s.check(capi, given=[12, 60, 1, 0, 4])
    s.check(capi, given=[-3, 1000, 0, 7, 4])                            # at least one, at most all


def test_pages_that_are_not_there(capi):
    s = Step(8, [5, 20, 40], [40, 40, 64], agree=1.0)
    s.table[0, 1], s.table[1, 2] = -1, 10 ** 6
    s.check(capi)
    s = Step(9, [5, 20, 40], [40, 40, 64], agree=1.0)
    s.table = np.ascontiguousarray(s.table[:, :3])                      # a table that ends before the request
    s.check(capi)
    s = Step(10, [0, 0], [40, 30], agree=1.0)
    s.lens = np.array([20, 0])                                          # shorter than their nodes
    s.check(capi)


def test_the_same_token_twice_and_a_choice_that_nobody_drafted(capi):
    s = Step(11, [3, 3], [6, 4], kinds=("star",))
    s.tokens[:], s.picked[:] = 4, 4
    s.picked[6] = 5
    assert s.check(capi).tolist() == [2, 1]


def test_one_layer_and_rows_of_no_request(capi):
    s = Step(12, [3, 30], [20, 30])
    s.check(capi, whole=False)
    pad = lambda x, v: np.concatenate([np.full(3, v), x, np.full(5, v)])
    s.parents, s.tokens, s.picked, s.starts = pad(s.parents, 0), pad(s.tokens, 1), pad(s.picked, 1), s.starts + 3
    s.check(capi)


def test_a_captured_step_is_replayed(capi):
    s = Step(13, [9, 50], [30, 40])
    put = lambda x, t: torch.tensor(np.asarray(x), dtype=t, device=DEV)
    cache, scales = put(s.cache, torch.uint8), put(s.scales, torch.uint8)
    args = [put(s.table, torch.int32), put(s.starts, torch.int32), put(s.lens, torch.int32), put(s.parents, torch.int32)]
    tokens, picked = put(s.tokens, torch.int64), put(s.picked, torch.int64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        capi.page_keep(cache, scales, *args, tokens, picked)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = capi.page_keep(cache, scales, *args, tokens, picked)
    for turn in range(4):
        t, p = s.rng.integers(0, 3, len(s.tokens)), s.rng.integers(0, 3, len(s.tokens))
        cache.copy_(put(s.cache, torch.uint8)), scales.copy_(put(s.scales, torch.uint8))
        tokens.copy_(put(t, torch.int64)), picked.copy_(put(p, torch.int64))
        graph.replay()
        held = s.cache.copy(), s.scales.copy()
        for g, w in zip(got, paged_more.keep(*held, s.table, s.starts, s.lens, s.parents, t, p)):
            assert np.array_equal(g.cpu().numpy(), w), turn
        assert np.array_equal(cache.cpu().numpy(), held[0]) and np.array_equal(scales.cpu().numpy(), held[1])


def test_refusals(capi):
    s = Step(14, [9], [5])
    put = lambda x, t: torch.tensor(np.asarray(x), dtype=t, device=DEV)
    cache, scales = put(s.cache, torch.uint8), put(s.scales, torch.uint8)
    base = dict(cache=cache, scales=scales, block_table=put(s.table, torch.int32), query_starts=put(s.starts, torch.int32),
                kv_lens=put(s.lens, torch.int32), parents=put(s.parents, torch.int32), tokens=put(s.tokens, torch.int64),
                picked=put(s.picked, torch.int64))
    for text, change in (("one type", dict(tokens=base["tokens"].int())), ("each of 5 nodes", dict(picked=base["picked"][:4])),
                         ("given must", dict(given=put([1, 1], torch.int32))), ("given must", dict(given=put([1], torch.int64))),
                         ("int32", dict(parents=base["parents"].long())), ("one entry more", dict(kv_lens=put([14, 3], torch.int32))),
                         ("has 2 requests", dict(block_table=base["block_table"].repeat(2, 1))),
                         ("scales must", dict(scales=scales[:1])), ("layers overlap", dict(cache=cache[:1].expand_as(cache))),
                         ("CUDA", dict(tokens=base["tokens"].cpu())), ("64, 128 or 256", dict(cache=cache[..., :16]))):
        with pytest.raises(RuntimeError, match=text):
            capi.page_keep(**{**base, **change})
    assert np.array_equal(cache.cpu().numpy(), s.cache)
