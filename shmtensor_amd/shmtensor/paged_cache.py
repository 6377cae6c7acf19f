"""Keys and values of the requests that a language model is answering, in pages in HBM, 4 or 8 bits a value: the bookkeeping
around the operators page_plan, page_set, page_fetch, page_attention, page_tree and page_keep (include/shmt.h says what those
compute).

    cache = PagedCache(pages=4096, layers=32, kv_heads=8, dim=128, requests=64, max_len=32768)
    step = cache.plan([17, 1, 0, 1])          # new tokens of each request in this step
    for layer in range(32):
        cache.set(step, layer, keys, values)            # [step.tokens, kv_heads, dim], request by request
        out = cache.attend(step, layer, query)          # [step.tokens, heads, dim]
    cache.release(1)                                    # request 1 is done: its pages are free again

Several drafted continuations at once, as trees (a node's parent is the index of one in front of it, or -1):

    step = cache.plan([5, 3, 0, 1], parents=[-1, 0, 0, 1, 1,  -1, 0, 1,  -1])
    ...                                                 # set and attend as above; step.positions are the nodes' places
    counts, path, token = cache.keep(step, tokens, picked)   # picked: the model's choice behind each node
    # request r holds counts[r] of its nodes now, the rows of those that agree with the model; token[r] comes next

A decoder's view of an encoder's states, which are planned and set once, like a prompt:

    out = states.attend_all(layer, query, query_starts, max_query_len=5)

The reference has no counterpart: its caches hold feature rows bit for bit under slots from a hash map
(src/cache_feature_set.cu, src/cache_feature_fetch.cu).
"""
import numpy as np
import torch

from . import capi

_STEPS_AHEAD = 32


class Step:
    """One step's plan, all on the GPU but the counts: query_starts [requests + 1], kv_lens [requests], positions and
    slots [tokens]; tokens; max_query_len. Of a step over trees also the parents and the numbered nodes [tokens, 4]."""

    def __init__(self, query_starts, kv_lens, positions, slots, max_query_len, new, parents=None, nodes=None):
        self.query_starts, self.kv_lens, self.positions, self.slots = query_starts, kv_lens, positions, slots
        self.tokens, self.max_query_len = positions.numel(), max_query_len
        self.new, self.parents, self.nodes = new, parents, nodes


class PagedCache:
    """`requests` places for requests of up to `max_len` tokens, sharing `pages` pages of `page` tokens. All layers use
    the same block table. The host keeps the requests' lengths and how many pages are free, so that no step waits for
    the GPU (until it is _STEPS_AHEAD steps behind); which pages they are is known to the GPU only."""

    def __init__(self, pages, kv_heads, dim, requests, max_len, layers=1, page=16, device="cuda", bits=4):
        if bits not in (4, 8):
            raise ValueError("a value is held in 4 or 8 bits, not %r" % (bits,))
        self.page, self.max_len, self.bits = page, max_len, bits
        width = -(-max_len // page)
        # a page's layers side by side would be as good; this keeps each layer's pages together
        self.cache = torch.zeros((layers, pages, kv_heads, 2, page, dim * bits // 8), dtype=torch.uint8, device=device)
        if bits == 8:
            self.cache = self.cache.view(torch.float8_e4m3fn)
        self.scales = torch.zeros((layers, pages, kv_heads, 2, dim // 32, page), dtype=torch.uint8, device=device)
        self.block_table = torch.full((requests, width), -1, dtype=torch.int32, device=device)
        self.lens = np.zeros(requests, dtype=np.int64)
        self._dropped = [(0, 0)] * requests          # pages [from, to) of a request that trim() gave back
        self._drafted = np.zeros(requests, dtype=np.int64)   # new tokens that keep() may still take back
        self._open = None                            # the step over trees that keep() may end
        self._gone = set()                           # requests that were released since it was planned
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

    def plan(self, new_lens, parents=None):
        """Pages and slots for new_lens[r] further tokens of every request r (host integers). Raises RuntimeError, and
        changes nothing, if there are not enough free pages or a request grows beyond max_len. With parents, one for each new
        token, the requests' new tokens are trees: keep() ends such a step. (An int32 tensor on the GPU; host integers are
        copied there, which waits for what is queued.) A step over trees that is not ended before the next plan() stays whole:
        its nodes are text from then on, one behind the other."""
        new = np.asarray(new_lens, dtype=np.int64).copy()    # the step and trim() go by it until keep()
        if new.shape != self.lens.shape or (new < 0).any():
            raise ValueError("new_lens must hold a length >= 0 for each of %d requests" % len(self.lens))
        total = self.lens + new
        if (total > self.max_len).any():
            raise RuntimeError("request %d grows beyond max_len = %d" % (int((total > self.max_len).argmax()), self.max_len))
        need = int((self._pages(total) - self._pages(self.lens)).sum())
        if need > self.free_pages:
            raise RuntimeError("%d pages needed, %d free" % (need, self.free_pages))
        if parents is not None:
            if len(new) >= 1 << 24:
                raise ValueError("a step over trees has less than 2^24 requests, as keep() does")
            parents = torch.as_tensor(parents, dtype=torch.int32)
            if parents.shape != (int(new.sum()),):
                raise ValueError("parents must hold an entry for each of %d new tokens" % new.sum())
            parents = parents.to(self._free.device, copy=True)    # keep() follows them
        device_new = self._to_device(new)
        starts, kv_lens, positions, slots, _ = capi.page_plan(self._kv_lens, device_new, self.block_table, self._free,
                                                              self.page, int(new.sum()))
        self._free, self._kv_lens, self.lens = self._free[need:], kv_lens, total
        nodes = None
        self._drafted = np.zeros_like(new)
        if parents is not None:
            nodes, positions = capi.page_tree(parents, starts, kv_lens)
            self._drafted = new
        step = Step(starts, kv_lens, positions, slots, int(new.max(initial=0)), new, parents, nodes)
        self._open, self._gone = step if parents is not None else None, set()
        return step

    def set(self, step, layer, keys, values):
        """Rounds the step's keys and values [tokens, kv_heads, dim] into the cache."""
        capi.page_set(self.cache[layer], self.scales[layer], step.slots, keys, values)

    def fetch(self, step, layer, dtype):
        """[keys, values] of the step's tokens as the cache holds them."""
        return capi.page_fetch(self.cache[layer], self.scales[layer], step.slots, dtype)

    def attend(self, step, layer, query, softmax_scale=None, window=0, sinks=0, return_lse=False):
        """Attention of the step's queries [tokens, heads, dim] over what the cache holds for their requests; with a
        window, over the last `window` tokens and the first `sinks`. In a step over trees a node sees what was there before
        the step, itself and the nodes above it."""
        return capi.page_attention(query, self.cache[layer], self.scales[layer], self.block_table, step.query_starts,
                                   step.kv_lens, softmax_scale, window=window, sinks=sinks,
                                   max_query_len=step.max_query_len, return_lse=return_lse, tree=step.nodes)

    def attend_all(self, layer, query, query_starts, max_query_len=0, softmax_scale=None, return_lse=False):
        """Attention of queries [tokens, heads, dim], request r's from query_starts[r] on (int32 on the GPU, requests + 1
        entries), over all that the cache holds for their requests: a decoder's over an encoder's states. max_query_len:
        the most queries of a request, if known."""
        return capi.page_attention(query, self.cache[layer], self.scales[layer], self.block_table, query_starts,
                                   self._kv_lens, softmax_scale, max_query_len=max_query_len, return_lse=return_lse,
                                   causal=False)

    def keep(self, step, tokens, picked, given=None):
        """Ends the step over trees that plan() made last: of each request's nodes those stay along which `picked` (the
        model's choice behind each node) agrees with `tokens`, both [step.tokens] on the GPU; their rows are moved together
        in all layers, the places and pages behind them are free again. given (int32 on the GPU): how many of a request's
        first nodes are no drafts (default 1). Returns (counts, path, token): counts (host integers) nodes of each request
        that stay; path [step.tokens] their indices, then -1; token [requests] what was picked behind the last of them. Of a
        request that was released since plan() nothing stays: its count is 0, its path and token are -1.
        Waits for the GPU: the counts are the requests' new lengths."""
        if step.parents is None:
            raise ValueError("the step has no trees: plan() was called without parents")
        if step is not self._open:
            raise ValueError("the step is not the last one that was planned, or it has been ended")
        counts, path, token = capi.page_keep(self.cache, self.scales, self.block_table, step.query_starts, step.kv_lens,
                                             step.parents, tokens, picked, given)
        kept = counts.cpu().numpy().astype(np.int64)
        before = self.lens - step.new
        self._kv_lens = step.kv_lens - (step.query_starts[1:] - step.query_starts[:-1]) + counts
        ends = np.cumsum(step.new)
        for r in self._gone:                         # (it has no pages: nothing of it was moved)
            before[r] = kept[r] = 0
            self._kv_lens[r:r + 1].zero_()
            path[int(ends[r] - step.new[r]):int(ends[r])].fill_(-1)
            token[r:r + 1].fill_(-1)
        held, need = self._pages(self.lens), self._pages(before + kept)
        self.lens, self._drafted = before + kept, np.zeros_like(kept)
        self._open, self._gone = None, set()
        spans = [(r, int(need[r]), int(held[r])) for r in np.nonzero(need < held)[0]]
        if spans:
            at = np.concatenate([r * self.block_table.shape[1] + np.arange(a, b) for r, a, b in spans])
            at = torch.from_numpy(at).to(self._free.device)
            flat, n = self.block_table.view(-1), self.free_pages
            free = self._free.new_empty(n + len(at))
            free[:n].copy_(self._free)
            free[n:].copy_(flat[at])
            self._free = free
            flat[at] = -1
        return kept, path, token

    def _give_back(self, request, first, end):
        if first < end:
            pages, n = self.block_table[request, first:end], self.free_pages
            free = self._free.new_empty(n + end - first)     # (torch.cat pins memory for its arguments, and may wait for that)
            free[:n].copy_(self._free)
            free[n:].copy_(pages)
            self._free = free
            pages.fill_(-1)

    def release(self, request):
        """The request is done; its place is empty again, for the next plan() to fill."""
        request = range(len(self.lens))[request]
        a, b = self._dropped[request]
        self._give_back(request, 0, a)
        self._give_back(request, b, self._pages(int(self.lens[request])))
        self._dropped[request] = (0, 0)
        self.lens = self.lens.copy()
        self.lens[request] = 0
        self._drafted = self._drafted.copy()
        self._drafted[request] = 0
        self._gone.add(request)
        self._kv_lens = self._kv_lens.clone()        # a step that is still in use keeps its own
        self._kv_lens[request:request + 1].zero_()

    def trim(self, request, window, sinks=0):
        """Gives back the pages that no further query of the request can see with this window and these sinks."""
        request = range(len(self.lens))[request]
        if window <= 0:
            return
        a, b = self._dropped[request]
        first = self._pages(sinks) if b == 0 else a
        end = max(int(self.lens[request] - self._drafted[request]) + 1 - window, 0) // self.page
        if first >= end:
            return
        if b == 0:
            self._give_back(request, first, end)
        else:
            self._give_back(request, b, end)
        self._dropped[request] = (first, max(end, b))
