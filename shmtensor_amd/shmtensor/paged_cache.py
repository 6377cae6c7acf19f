"""Keys and values of the requests that a language model is answering, in pages in HBM, 4 bits a value: the bookkeeping
around the operators page_plan, page_set, page_fetch and page_attention (include/shmt.h says what those compute).

    cache = PagedCache(pages=4096, layers=32, kv_heads=8, dim=128, requests=64, max_len=32768)
    step = cache.plan([17, 1, 0, 1])          # new tokens of each request in this step
    for layer in range(32):
        cache.set(step, layer, keys, values)            # [step.tokens, kv_heads, dim], request by request
        out = cache.attend(step, layer, query)          # [step.tokens, heads, dim]
    cache.release(1)                                    # request 1 is done: its pages are free again

The reference has no counterpart: its caches hold feature rows bit for bit under slots from a hash map
(src/cache_feature_set.cu, src/cache_feature_fetch.cu).
"""
import numpy as np
import torch

from . import capi

_STEPS_AHEAD = 32


class Step:
    """One step's plan, all on the GPU but the counts: query_starts [requests + 1], kv_lens [requests], positions and
    slots [tokens]; tokens; max_query_len."""

    def __init__(self, query_starts, kv_lens, positions, slots, max_query_len):
        self.query_starts, self.kv_lens, self.positions, self.slots = query_starts, kv_lens, positions, slots
        self.tokens, self.max_query_len = positions.numel(), max_query_len


class PagedCache:
    """`requests` places for requests of up to `max_len` tokens, sharing `pages` pages of `page` tokens. All layers use
    the same block table. The host keeps the requests' lengths and how many pages are free, so that no step waits for
    the GPU (until it is _STEPS_AHEAD steps behind); which pages they are is known to the GPU only."""

    def __init__(self, pages, kv_heads, dim, requests, max_len, layers=1, page=16, device="cuda"):
        self.page, self.max_len = page, max_len
        width = -(-max_len // page)
        # a page's layers side by side would be as good; this keeps each layer's pages together
        self.cache = torch.zeros((layers, pages, kv_heads, 2, page, dim // 2), dtype=torch.uint8, device=device)
        self.scales = torch.zeros((layers, pages, kv_heads, 2, dim // 32, page), dtype=torch.uint8, device=device)
        self.block_table = torch.full((requests, width), -1, dtype=torch.int32, device=device)
        self.lens = np.zeros(requests, dtype=np.int64)
        self._dropped = [(0, 0)] * requests          # pages [from, to) of a request that trim() gave back
        self._free = torch.arange(pages, dtype=torch.int32, device=device)
        self._kv_lens = torch.zeros(requests, dtype=torch.int32, device=device)
        # New lengths on their way to the GPU: from memory that is not pinned a copy waits for all that is queued, and so does
        # pinning memory. A place is written again when its copy has run.
        self._staging = torch.empty((_STEPS_AHEAD, requests), dtype=torch.int32, pin_memory=True)
        self._copied = [None] * _STEPS_AHEAD
        self._turn = 0

    @property
    def free_pages(self):
        return self._free.numel()

    def _pages(self, tokens):
        return -(-tokens // self.page)

    def _to_device(self, lens):
        at = self._turn = (self._turn + 1) % _STEPS_AHEAD
        if self._copied[at] is None:
            self._copied[at] = torch.cuda.Event()
        else:
            self._copied[at].synchronize()
        self._staging[at].numpy()[:] = lens
        there = self._staging[at].to(self._free.device, non_blocking=True)
        self._copied[at].record()
        return there

    def plan(self, new_lens):
        """Pages and slots for new_lens[r] further tokens of every request r (host integers). Raises RuntimeError, and
        changes nothing, if there are not enough free pages or a request grows beyond max_len."""
        new = np.asarray(new_lens, dtype=np.int64)
        if new.shape != self.lens.shape or (new < 0).any():
            raise ValueError("new_lens must hold a length >= 0 for each of %d requests" % len(self.lens))
        total = self.lens + new
        if (total > self.max_len).any():
            raise RuntimeError("request %d grows beyond max_len = %d" % (int((total > self.max_len).argmax()), self.max_len))
        need = int((self._pages(total) - self._pages(self.lens)).sum())
        if need > self.free_pages:
            raise RuntimeError("%d pages needed, %d free" % (need, self.free_pages))
        device_new = self._to_device(new)
        starts, kv_lens, positions, slots, _ = capi.page_plan(self._kv_lens, device_new, self.block_table, self._free,
                                                              self.page, int(new.sum()))
        self._free, self._kv_lens, self.lens = self._free[need:], kv_lens, total
        return Step(starts, kv_lens, positions, slots, int(new.max(initial=0)))

    def set(self, step, layer, keys, values):
        """Rounds the step's keys and values [tokens, kv_heads, dim] into the cache."""
        capi.page_set(self.cache[layer], self.scales[layer], step.slots, keys, values)

    def fetch(self, step, layer, dtype):
        """[keys, values] of the step's tokens as the cache holds them."""
        return capi.page_fetch(self.cache[layer], self.scales[layer], step.slots, dtype)

    def attend(self, step, layer, query, softmax_scale=None, window=0, sinks=0, return_lse=False):
        """Attention of the step's queries [tokens, heads, dim] over what the cache holds for their requests; with a
        window, over the last `window` tokens and the first `sinks`."""
        return capi.page_attention(query, self.cache[layer], self.scales[layer], self.block_table, step.query_starts,
                                   step.kv_lens, softmax_scale, window=window, sinks=sinks,
                                   max_query_len=step.max_query_len, return_lse=return_lse)

    def _give_back(self, request, first, end):
        if first < end:
            pages, n = self.block_table[request, first:end], self.free_pages
            free = self._free.new_empty(n + end - first)     # (torch.cat pins memory for its arguments, and may wait for that)
            free[:n].copy_(self._free)
            free[n:].copy_(pages)
            self._free = free
            pages.fill_(-1)

    def release(self, request):
        """The request is done; its place is empty again."""
        a, b = self._dropped[request]
        self._give_back(request, 0, a)
        self._give_back(request, b, self._pages(int(self.lens[request])))
        self._dropped[request] = (0, 0)
        self.lens[request] = 0
        self._kv_lens = self._kv_lens.clone()        # a step that is still in use keeps its own
        self._kv_lens[request:request + 1].zero_()

    def trim(self, request, window, sinks=0):
        """Gives back the pages that no further query of the request can see with this window and these sinks."""
        if window <= 0:
            return
        a, b = self._dropped[request]
        first = self._pages(sinks) if b == 0 else a
        end = max(int(self.lens[request]) + 1 - window, 0) // self.page
        if first >= end:
            return
        if b == 0:
            self._give_back(request, first, end)
        else:
            self._give_back(request, b, end)
        self._dropped[request] = (first, max(end, b))
