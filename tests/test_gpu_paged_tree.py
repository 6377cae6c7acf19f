"""Trees of drafted tokens numbered (page_tree): whole numbers, equal to the definition's (oracle/paged_more.py)."""
import numpy as np
import pytest
import torch

from oracle import paged_more

pytestmark = pytest.mark.gpu
DEV = "cuda"


def grown(rng, n, kind):
    """Parents of a tree of n nodes."""
    if kind == "chain":
        return np.arange(n) - 1
    if kind == "star":
        return np.minimum(np.arange(n) - 1, 0)
    if kind == "forest":
        return np.where(rng.random(n) < 0.3, -1, (rng.random(n) * np.arange(n)).astype(int) - (np.arange(n) == 0))
    if kind == "late":                                                  # long, with short branches
        return np.maximum(np.arange(n) - 1 - (rng.random(n) < 0.3) * rng.integers(0, 4, n), -1)
    return np.where(np.arange(n) == 0, -1, (rng.random(n) * np.arange(n)).astype(int))


def _check(capi, parents, starts, lens, dtype=torch.int32):
    put = lambda x, t: torch.tensor(np.asarray(x), dtype=t, device=DEV)
    nodes, positions = capi.page_tree(put(parents, torch.int32), put(starts, dtype), put(lens, dtype))
    want = paged_more.tree(parents, starts, lens)
    assert nodes.dtype == positions.dtype == torch.int32
    assert np.array_equal(nodes.cpu().numpy(), want[0]) and np.array_equal(positions.cpu().numpy(), want[1])


@pytest.mark.parametrize("kind", ["tree", "chain", "star", "forest", "late"])
@pytest.mark.parametrize("n", [1, 2, 3, 31, 63, 64, 65, 127, 128, 129, 500, 1024, 1025, 1500])
def test_one_request(capi, kind, n):
    rng = np.random.default_rng(n)
    _check(capi, grown(rng, n, kind), [0, n], [n + 17])


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_many_requests(capi, dtype):
    rng = np.random.default_rng(7)
    kinds = ["tree", "chain", "star", "forest", "late"]
    news = np.concatenate([rng.integers(0, 65, 300), [0, 0, 200, 64, 65, 1, 900, 0, 3], rng.integers(0, 12, 200), [1100, 0]])
    parents = [grown(rng, n, kinds[i % 5]) for i, n in enumerate(news)]
    starts = np.concatenate([[0], np.cumsum(news)])
    _check(capi, np.concatenate(parents), starts, news + rng.integers(0, 5000, len(news)), dtype)


def test_rows_of_no_request_and_none_at_all(capi):
    rng = np.random.default_rng(8)
    parents = np.concatenate([[5, 5, 5], grown(rng, 9, "tree"), grown(rng, 80, "late"), [0, 1]])
    _check(capi, parents, [3, 12, 92], [20, 30])                        # a request shorter than its nodes, too
    _check(capi, parents, [0], [])
    _check(capi, [], [0, 0], [4])
    _check(capi, [], [0], [])


def test_parents_that_are_none(capi):
    """Whatever lies not in front of its child is no parent."""
    rng = np.random.default_rng(9)
    for n in (40, 300):
        parents = grown(rng, n, "tree")
        parents[5], parents[7], parents[9], parents[20] = 5, 8, -7, 2 ** 31 - 1
        _check(capi, parents, [0, n], [n])


def test_a_captured_plan_is_replayed(capi):
    rng = np.random.default_rng(10)
    starts = torch.tensor([0, 30, 130], dtype=torch.int32, device=DEV)
    lens = torch.tensor([50, 130], dtype=torch.int32, device=DEV)
    parents = torch.zeros(130, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        capi.page_tree(parents, starts, lens)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nodes, positions = capi.page_tree(parents, starts, lens)
    for turn in range(4):
        now = np.concatenate([grown(rng, 30, "tree"), grown(rng, 100, ["late", "chain"][turn % 2])])
        parents.copy_(torch.from_numpy(now))
        lens.copy_(torch.tensor([50 + turn, 130 * turn]))
        graph.replay()
        want = paged_more.tree(now, [0, 30, 130], lens.tolist())
        assert np.array_equal(nodes.cpu().numpy(), want[0]) and np.array_equal(positions.cpu().numpy(), want[1])
        eager = capi.page_tree(parents, starts, lens)
        assert torch.equal(eager[0], nodes) and torch.equal(eager[1], positions)


def test_refusals(capi):
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    for bad, text in ((lambda: capi.page_tree(ints(0, 0).long(), ints(0, 2), ints(2)), "int32"),
                      (lambda: capi.page_tree(ints(0, 0).cpu(), ints(0, 2), ints(2)), "CUDA"),
                      (lambda: capi.page_tree(ints(0, 0)[None], ints(0, 2), ints(2)), "one-dimensional"),
                      (lambda: capi.page_tree(ints(0, 0), ints(0, 2), ints(2).long()), "one type"),
                      (lambda: capi.page_tree(ints(0, 0), ints(0, 2, 2), ints(2)), "one entry more"),
                      (lambda: capi.page_tree(ints(0, 0), ints(0, 2).float(), ints(2).float()), "int")):
        with pytest.raises(RuntimeError, match=text):
            bad()


def test_starts_that_descend(capi):
    """Requests whose rows overlap get words without a meaning, at their own rows only, and the call ends."""
    rng = np.random.default_rng(11)
    last = grown(rng, 100, "late")
    parents = np.concatenate([grown(rng, 2000, "tree"), grown(rng, 500, "star"), last])
    put = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    for _ in range(3):
        nodes, positions = capi.page_tree(put(parents), put([0, 2000, 500, 2500, 2600]), put([2000, 7, 2500, 130]))
        want = paged_more.tree(last, [0, 100], [130])
        assert np.array_equal(nodes[2500:].cpu().numpy(), want[0])
        assert np.array_equal(positions[2500:].cpu().numpy(), want[1])
