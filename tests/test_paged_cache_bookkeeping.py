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
