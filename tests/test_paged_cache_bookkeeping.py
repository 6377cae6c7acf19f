"""PagedCache's bookkeeping of lengths and pages, with the operators' definitions (oracle/) in the operators' place, so without a
GPU: what a caller does with its own arrays between the calls of a step, and the order of those calls."""
import types

import numpy as np
import pytest
import torch

from oracle import paged, paged_more


class _Event:
    def record(self):
        pass

    def synchronize(self):
        pass


class _HostTorch:
    """torch, but for pinned memory and events, which there are none of without a GPU."""
    cuda = types.SimpleNamespace(Event=_Event)

    def __getattr__(self, name):
        return getattr(torch, name)

    @staticmethod
    def empty(*args, pin_memory=False, **kw):
        return torch.empty(*args, **kw)


class _Definitions:
    @staticmethod
    def page_plan(cached, new, table, free, page, max_tokens):
        return [torch.from_numpy(x) for x in paged.plan(cached.numpy(), new.numpy(), table.numpy(), free.numpy(), page, max_tokens)]

    @staticmethod
    def page_tree(parents, starts, lens):
        return [torch.from_numpy(x).int() for x in paged_more.tree(parents.numpy(), starts.numpy(), lens.numpy())]

    @staticmethod
    def page_keep(cache, scales, table, starts, lens, parents, tokens, picked, given=None):
        counts, path, after = paged_more.keep(cache.numpy(), scales.numpy(), table.numpy(), starts.numpy(), lens.numpy(),
                                              parents.numpy(), tokens.numpy(), picked.numpy(), given)
        return torch.from_numpy(counts).int(), torch.from_numpy(path).int(), torch.from_numpy(after)


@pytest.fixture
def host_cache(capi, monkeypatch):
    from shmtensor_amd.shmtensor import paged_cache
    monkeypatch.setattr(paged_cache, "capi", _Definitions)
    monkeypatch.setattr(paged_cache, "torch", _HostTorch())
    return lambda **kw: paged_cache.PagedCache(**{**dict(pages=40, kv_heads=1, dim=64, requests=3, max_len=160, device="cpu"), **kw})


def _in_order(cache, lens, pages=40):
    """The host's lengths are the GPU's, every page has one owner, and a request has those that its length needs (no windows here)."""
    assert cache.lens.tolist() == list(lens) and cache._kv_lens.tolist() == list(lens)
    held = [[int(p) for p in row if p >= 0] for row in cache.block_table]
    assert [len(h) for h in held] == [-(-n // cache.page) for n in lens]
    assert sorted(sum(held, cache._free.tolist())) == list(range(pages)), "a page is lost or has two owners"


def test_lengths_are_the_callers_own(host_cache):
    """A caller's array of new lengths may be filled anew as soon as plan() has returned."""
    for buffer in (np.zeros(3, np.int64), np.zeros(3, np.int32), torch.zeros(3, dtype=torch.int64)):
        cache = host_cache()
        buffer[0], buffer[1], buffer[2] = 40, 33, 0
        cache.plan(buffer)
        buffer[0], buffer[1], buffer[2] = 20, 5, 1
        step = cache.plan(buffer, parents=[-1, 0] + [1] * 18 + [-1, 0, 1, 2, 3] + [-1])
        buffer[0] = buffer[1] = buffer[2] = 1
        cache.trim(0, window=41)                                        # 40 tokens stay, whichever of the drafts do: all are in the window
        assert (cache.block_table[0, :4] >= 0).all()
        tokens, picked = torch.ones(26, dtype=torch.int64), torch.ones(26, dtype=torch.int64)
        picked[1] = 5                                                   # request 0: two nodes stay
        counts, _, _ = cache.keep(step, tokens, picked)
        assert counts.tolist() == [2, 5, 1]
        _in_order(cache, [42, 38, 1])


def test_parents_are_the_callers_own(host_cache):
    """So may the tensor of parents: the step keeps what it was planned with."""
    cache = host_cache()
    parents = torch.tensor([-1, 0, 1, 2, -1, 0], dtype=torch.int32)
    step = cache.plan([4, 2, 0], parents=parents)
    parents.fill_(-1)
    ones = torch.ones(6, dtype=torch.int64)
    counts, path, _ = cache.keep(step, ones, ones)
    assert counts.tolist() == [4, 2, 0] and path.tolist() == [0, 1, 2, 3, 0, 1]
    _in_order(cache, [4, 2, 0])


def test_a_request_is_released_while_its_step_runs(host_cache):
    """Its pages are free at once; the step ends for the others, and keeps nothing of the one that is gone."""
    for gone in ([1], [0, 2], [0, 1, 2], [1, 1]):
        cache = host_cache()
        cache.plan([40, 16, 30])
        parents = [-1, 0, 0, 2] + [-1, 0, 1] + [-1, 0, 1, 2, 3]
        step = cache.plan([4, 3, 5], parents=parents)
        for r in gone:
            cache.release(r)
        assert cache.lens.tolist() == [0 if r in gone else n for r, n in enumerate((44, 19, 35))]
        tokens = torch.tensor([7, 8, 9, 7] + [7, 7, 7] + [1, 2, 3, 4, 5])
        picked = torch.tensor([9, 5, 7, 6] + [7, 7, 4] + [2, 3, 6, 6, 6])
        counts, path, token = cache.keep(step, tokens, picked)
        want = [(3, [0, 2, 3, -1], 6), (3, [0, 1, 2], 4), (3, [0, 1, 2, -1, -1], 6)]
        want = [(0, [-1] * len(p), -1) if r in gone else (n, p, t) for r, (n, p, t) in enumerate(want)]
        assert counts.tolist() == [n for n, _, _ in want]
        assert path.tolist() == sum((p for _, p, _ in want), []) and token.tolist() == [t for _, _, t in want]
        lens = [0 if r in gone else n for r, n in enumerate((43, 19, 33))]
        _in_order(cache, lens)
        with pytest.raises(ValueError, match="not the last one"):
            cache.keep(step, tokens, picked)
        step = cache.plan([1, 20, 1])                                   # the places serve on
        assert step.kv_lens.tolist() == [lens[0] + 1, lens[1] + 20, lens[2] + 1]
        _in_order(cache, step.kv_lens.tolist())


def test_a_step_that_is_never_ended_stays_whole(host_cache):
    """The next plan() takes all of its nodes for the requests' text."""
    cache = host_cache()
    cache.plan([10, 0, 3])
    step = cache.plan([3, 2, 0], parents=[-1, 0, 0, -1, 0])
    with pytest.raises(RuntimeError, match="beyond max_len"):
        cache.plan([150, 150, 150])                                     # refused: the step is still the last one
    assert cache.keep(step, torch.ones(5, dtype=torch.int64), torch.zeros(5, dtype=torch.int64))[0].tolist() == [1, 1, 0]
    step = cache.plan([3, 2, 0], parents=[-1, 0, 0, -1, 0])
    after = cache.plan([1, 1, 1])
    assert after.positions.tolist() == [14, 3, 3] and after.kv_lens.tolist() == [15, 4, 4]
    with pytest.raises(ValueError, match="not the last one"):
        cache.keep(step, torch.ones(5, dtype=torch.int64), torch.ones(5, dtype=torch.int64))
    _in_order(cache, [15, 4, 4])


def test_requests_counted_from_the_end(host_cache):
    """release(-1) and trim(-1) mean the last request, lengths on the GPU included; a request that there is not is refused."""
    cache = host_cache()
    cache.plan([40, 16, 100])
    cache.trim(-1, window=20)
    assert (cache.block_table[2] >= 0).sum() == 2 and cache._dropped[2] == (0, 5)
    cache.release(-1)
    assert cache._kv_lens.tolist() == [40, 16, 0]
    cache.plan([1, 1, 30])
    _in_order(cache, [41, 17, 30])
    for wrong in (3, -4):
        with pytest.raises(IndexError):
            cache.release(wrong)
        with pytest.raises(IndexError):
            cache.trim(wrong, window=1)
    _in_order(cache, [41, 17, 30])


def test_more_requests_than_a_step_over_trees_may_have(host_cache):
    """Refused before the step, not at its end."""
    cache = host_cache(requests=1 << 24, max_len=16)
    new = np.zeros(1 << 24, np.int64)
    with pytest.raises(ValueError, match="2\\^24"):
        cache.plan(new, parents=[])
    assert cache.free_pages == 40 and not cache.lens.any()
