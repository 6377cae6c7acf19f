"""Attention over the paged cache with other rules of what a row sees than a chain's (trees of drafted tokens; all of an
encoder's states) and over caches in 8 bits, against the definition in 64 bits (oracle/paged_more.py). The bounds are those of
test_gpu_paged_attention.py: nothing in them depends on which tokens a row sees or how many bits hold a value, both of which
become bfloat16 exactly."""
import numpy as np
import pytest
import torch

from oracle import paged_more
from test_gpu_paged_attention import _close
from test_gpu_paged_tree import grown

pytestmark = pytest.mark.gpu
DEV = "cuda"
KINDS = ("tree", "late", "chain", "star", "forest")


class Batch:
    """Requests in a cache whose other places hold garbage: pages of no request, places behind a request's end."""

    def __init__(self, seed, kv_lens, query_lens, heads, kv_heads, dim, page, dtype, bits=4, seen="causal", kinds=KINDS, spread=1.5):
        gen = torch.Generator().manual_seed(seed)
        rng = self.rng = np.random.default_rng(seed)
        kv_lens, query_lens = np.asarray(kv_lens), np.asarray(query_lens)
        count = -(-kv_lens // page)
        pages = int(count.sum()) + 3
        order = rng.permutation(pages)
        self.bits, self.seen = bits, seen
        self.cache = torch.randint(0, 256, (pages, kv_heads, 2, page, dim * bits // 8), generator=gen, dtype=torch.uint8)
        # garbage: blocks that are not numbers, and in 8 bits codes that are not
        self.scales = torch.where(torch.rand((pages, kv_heads, 2, dim // 32, page), generator=gen) < 0.5, 255, 127).byte()
        self.table = torch.full((len(kv_lens), max(1, int(count.max(initial=0)))), -1, dtype=torch.int32)
        at = 0
        base = 127 if bits == 4 else 120
        for b, n in enumerate(count):
            mine = order[at:at + n]
            at += n
            self.table[b, :n] = torch.from_numpy(mine).int()
            for i, p in enumerate(mine):
                live = min(page, int(kv_lens[b]) - i * page)
                self.scales[p, ..., :live] = torch.randint(base - 3, base + 1, (kv_heads, 2, dim // 32, live), generator=gen).byte()
                if bits == 8:                                          # normal numbers of about 1 to 64 times the scale
                    x = torch.randn((kv_heads, 2, live, dim), generator=gen) * 40
                    self.cache[p, :, :, :live] = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        self.starts = torch.tensor(np.concatenate([[0], np.cumsum(query_lens)]), dtype=torch.int32)
        self.kv_lens = torch.tensor(kv_lens, dtype=torch.int32)
        self.query = (torch.randn((int(self.starts[-1]), heads, dim), generator=gen) * spread).to(dtype)
        self.parents = np.concatenate([grown(rng, k, kinds[i % len(kinds)]) for i, k in enumerate(query_lens)] + [np.zeros(0, int)])
        self.scale = dim ** -0.5

    def args(self):
        q, c, s, t, i, l = [x.to(DEV) for x in (self.query, self.cache, self.scales, self.table, self.starts, self.kv_lens)]
        return [q, c.view(torch.float8_e4m3fn) if self.bits == 8 else c, s, t, i, l]

    def rule(self, capi):
        if self.seen == "tree":
            put = lambda x: torch.as_tensor(x).int().to(DEV)
            return dict(tree=capi.page_tree(put(self.parents), put(self.starts), put(self.kv_lens))[0])
        return dict(causal=self.seen == "causal")

    def want(self, **kw):
        return paged_more.attention(self.query.double().numpy(), self.cache.numpy(), self.scales.numpy(), self.table.numpy(),
                                    self.starts.numpy(), self.kv_lens.numpy(), self.scale, self.bits, self.seen, self.parents, **kw)


def _check(capi, b, **kw):
    hint = kw.pop("max_query_len", int(b.starts.diff().max()) if len(b.kv_lens) else 0)
    got, lse = capi.page_attention(*b.args(), b.scale, max_query_len=hint, return_lse=True, **b.rule(capi), **kw)
    _close(got, lse, b.want(**kw), b.query.dtype, b.query.shape[2])
    return got, lse


RULES = [(4, "tree"), (4, "all"), (8, "causal"), (8, "tree"), (8, "all")]
WINDOWS = [(0, 0), (1, 0), (7, 3), (33, 4), (100, 300)]


@pytest.mark.parametrize("bits, seen", RULES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (8, 2), (5, 5), (16, 1), (40, 1)])
def test_single_tokens(capi, bits, seen, dtype, dim, heads, kv_heads):
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 128, 129, 300, 0, 257]
    _check(capi, Batch(heads * dim, lens, [1] * len(lens), heads, kv_heads, dim, 16, dtype, bits, seen))


@pytest.mark.parametrize("bits, seen", RULES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_several_tokens(capi, bits, seen, dtype, dim, page):
    """Trees of all shapes, whole prompts among them; requests without new tokens."""
    lens, q = [1, 40, 77, 160, 9, 130, 300, 33, 90], [1, 40, 5, 31, 0, 64, 2, 17, 13]
    for heads, kv_heads in ((4, 2), (3, 1)):
        _check(capi, Batch(page + dim, lens, q, heads, kv_heads, dim, page, dtype, bits, seen))


@pytest.mark.parametrize("bits, seen", RULES)
@pytest.mark.parametrize("dtype, dim", [(torch.bfloat16, 64), (torch.float16, 64), (torch.bfloat16, 128), (torch.float16, 128),
                                        (torch.bfloat16, 256), (torch.float16, 256)])
def test_many_rows(capi, bits, seen, dtype, dim):
    """The kernel for many rows: by the rows there are, and by a hint that is too great."""
    b = Batch(dim, [700, 300, 5, 333], [290, 300, 5, 64], 6, 2, dim, 16, dtype, bits, seen)
    _check(capi, b)
    b = Batch(dim + 1, [1, 400, 77, 260, 500, 34, 150], [1, 1, 77, 50, 3, 0, 129], 9, 3, dim, 32, dtype, bits, seen)
    _check(capi, b, max_query_len=4000)


@pytest.mark.parametrize("bits, seen", [(4, "tree"), (8, "causal"), (8, "tree")])
@pytest.mark.parametrize("window, sinks", WINDOWS[1:] + [(64, 0), (16, 16), (100000, 5)])
@pytest.mark.parametrize("dtype, dim, page", [(torch.bfloat16, 128, 16), (torch.float16, 64, 32), (torch.bfloat16, 256, 64)])
def test_windows_and_sinks(capi, bits, seen, window, sinks, dtype, dim, page):
    lens, q = [1, 400, 77, 260, 500, 34, 150, 40], [1, 1, 77, 50, 3, 0, 129, 33]
    b = Batch(window + dim, lens, q, 6, 2, dim, page, dtype, bits, seen, kinds=("late", "tree", "chain"))
    _check(capi, b, window=window, sinks=sinks)
    _check(capi, b, window=window, sinks=sinks, max_query_len=4000)


@pytest.mark.parametrize("bits", [4, 8])
def test_windows_whose_first_tokens_are_nodes(capi, bits):
    """Nodes that lie behind the first `sinks` tokens but not their places, or the other way round."""
    for n, cached in ((60, 0), (200, 5), (300, 100)):
        for window, sinks in ((3, 20), (20, 110), (1, 4)):
            b = Batch(n + sinks, [cached + n, n], [n, n], 4, 1, 64, 16, torch.bfloat16, bits, "tree", kinds=("tree", "late"))
            _check(capi, b, window=window, sinks=sinks)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_chain_is_the_causal_rule(capi, dim):
    """With a tree that is a chain and without one, in both kernels and with windows: the same sums, though in other parts."""
    for q in (1, 7, 150):
        b = Batch(q + dim, [500, 260, 150], [q, q, q], 8, 2, dim, 16, torch.bfloat16, 4, "tree", kinds=("chain",))
        for kw in ({}, dict(window=90, sinks=3)):
            want = b.want(**kw)
            for rule in (b.rule(capi), {}):
                got, lse = capi.page_attention(*b.args(), b.scale, max_query_len=q, return_lse=True, **rule, **kw)
                _close(got, lse, want, torch.bfloat16, dim)


@pytest.mark.parametrize("bits, seen", RULES)
def test_pages_that_are_missing_are_not_seen(capi, bits, seen):
    for dim, q in ((128, 1), (64, 3), (256, 70), (128, 200)):
        b = Batch(dim + q, [500, 260, 300], [q, q, q], 4, 2, dim, 32, torch.bfloat16, bits, seen)
        b.table[0, 2:5] = -1
        b.table[1, :] = -1
        b.table[2, 0], b.table[2, 3] = len(b.cache), 2 ** 31 - 1
        _check(capi, b)


@pytest.mark.parametrize("bits, seen", RULES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_more_queries_than_tokens(capi, bits, seen, dim):
    b = Batch(5, [3, 0, 50], [9, 4, 60], 4, 1, dim, 16, torch.float16, bits, seen)
    got, lse = _check(capi, b)
    assert bool((got[9:13] == 0).all()) and bool(lse[9:13].isneginf().all())
    if seen != "all":
        _check(capi, b, window=5, sinks=2)


@pytest.mark.parametrize("bits, seen", RULES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_work_split_over_long_requests(capi, bits, seen, dtype):
    _check(capi, Batch(1, [9001], [1], 5, 1, 128, 32, dtype, bits, seen))
    _check(capi, Batch(2, [5, 6000, 1, 3000, 17], [1, 2, 1, 1, 3], 4, 2, 64, 16, dtype, bits, seen))
    _check(capi, Batch(3, [4100], [20], 8, 1, 256, 64, dtype, bits, seen))
    if seen != "all":
        _check(capi, Batch(4, [5000, 3], [40, 3], 4, 1, 128, 16, dtype, bits, seen), window=2500, sinks=70)


@pytest.mark.parametrize("bits, seen", RULES)
@pytest.mark.parametrize("dtype, dim", [(torch.bfloat16, 64), (torch.float16, 128), (torch.bfloat16, 256)])
@pytest.mark.parametrize("most, requests", [(7, 70), (260, 25)])
def test_shares_that_end_anywhere(capi, bits, seen, dtype, dim, most, requests):
    """Items of all lengths and fillings, so that shares of the work begin and end at every place of an item: within its tokens, at
    its end, behind it."""
    rng = np.random.default_rng(dim)
    lens = rng.integers(0, 900, requests)
    q = np.minimum(rng.integers(0, most + 1, requests), lens + (1 if seen == "all" else 0))
    heads, kv_heads = (12, 12) if most == 7 else (8, 4)
    b = Batch(dim, lens, q, heads, kv_heads, dim, 16, dtype, bits, seen)
    _check(capi, b)
    if seen != "all" and most == 7:
        _check(capi, b, window=300, sinks=20)


@pytest.mark.parametrize("bits, seen", [(4, "all"), (8, "causal"), (8, "all")])
@pytest.mark.parametrize("lens, queries", [([300, 40, 270], [4000, 5000, 1500]), ([300, 20], [9000, 9000]), ([30], [11000])])
def test_more_items_than_threads(capi, bits, seen, lens, queries):
    """600 and 1,100 items of 256 rows, which a workgroup's threads do not count at once."""
    _check(capi, Batch(sum(lens), lens, queries, 16, 1, 64, 16, torch.bfloat16, bits, seen))


@pytest.mark.parametrize("bits, seen", RULES)
@pytest.mark.parametrize("q", [1, 9, 100])
def test_not_a_number_where_it_is_seen_and_nowhere_else(capi, bits, seen, q):
    for dim in (64, 128, 256):
        b = Batch(dim, [200, 150], [q, q], 4, 2, dim, 16, torch.bfloat16, bits, seen, kinds=("tree", "late"))
        at = lambda r, j: int(b.table[r, j // 16])
        for j in {130, 120, 199, 200 - q // 2 - 1}:                    # one block of one value of head 0, of nodes, too
            b.scales[at(0, j), 0, 1, j % 2, j % 16] = 255
        b.scales[at(1, 149), 1, 0, 0, 149 % 16] = 255                  # a key that only the last row sees
        kw = {} if seen == "all" else dict(window=70)
        want = b.want(**kw)
        assert np.isnan(want[0]).any() and not np.isnan(want[0]).all()
        _check(capi, b, **kw)
        _check(capi, b, max_query_len=1000, **kw)


@pytest.mark.parametrize("bits, seen", [(8, "causal"), (8, "tree"), (4, "tree")])
@pytest.mark.parametrize("q", [3, 90])
def test_values_near_the_end_of_the_type(capi, bits, seen, q):
    """Values of 2^120 and more, which do not fit bfloat16's products, beside rows that do not see them."""
    for dim in (64, 128, 256):
        b = Batch(dim, [200, 150], [q, q], 4, 2, dim, 16, torch.bfloat16, bits, seen, kinds=("tree", "late"))
        at = lambda r, j: int(b.table[r, j // 16])
        byte = 247 if bits == 8 else 253
        for j in (198, 199, 197):
            page = at(0, j)
            b.scales[page, 1, 1, 0, j % 16] = byte
            codes = b.cache[page, 1, 1, j % 16]
            if bits == 8:
                codes[:32] = torch.tensor([0x38, 0xB8] * 16)           # 1 and -1: 2^120
            else:
                codes[:16] = 0xA2                                      # 1 and -1: 2^126
        got, lse = capi.page_attention(*b.args(), b.scale, max_query_len=q, return_lse=True, **b.rule(capi))
        want = b.want()
        _close(got, lse, want, torch.bfloat16, dim)


@pytest.mark.parametrize("bits, seen", RULES)
@pytest.mark.parametrize("rows", [1, 7, 200])
def test_extreme_scores(capi, bits, seen, rows):
    b = Batch(rows, [290, 100, 200], [min(rows, 90), 1, rows], 4, 2, 128, 16, torch.float16, bits, seen)
    big = b.scales[:, :, 0] != 255
    b.scales[:, :, 0][big] += 60
    for scale in (2.0 ** -60 * 128 ** -0.5, 0.0, -0.05 * 2.0 ** -60):
        b.scale = scale
        _check(capi, b)
    b = Batch(rows, [290, 100, 200], [min(rows, 90), 1, rows], 4, 2, 128, 16, torch.bfloat16, bits, seen)
    b.query[0] *= 2.0 ** 10
    b.query[-1] = 0
    _check(capi, b)


@pytest.mark.parametrize("bits, seen", RULES)
def test_rows_of_no_request_strides_and_widths(capi, bits, seen):
    b = Batch(7, [50, 60, 70], [1, 30, 2], 4, 2, 128, 16, torch.bfloat16, bits, seen)
    want = b.want()
    query, cache, scales, table, starts, lens = b.args()
    rule = b.rule(capi)
    padded = torch.cat([query[:7], query, query[:90]])
    if seen == "tree":
        put = lambda x: torch.as_tensor(x).int().to(DEV)
        rule = dict(tree=capi.page_tree(put(np.concatenate([np.full(7, 3), b.parents, np.zeros(33, int)])), starts + 7, lens)[0])

    wide = torch.full((3, 40), 1, dtype=torch.int32, device=DEV)
    wide[:, 4:4 + table.shape[1]] = table
    joint = torch.randn((len(padded), 10, 128), device=DEV).bfloat16()
    joint[:, 2:6] = padded
    for q, t, s, l in ((padded, table, starts, lens), (joint[:, 2:6], wide[:, 4:4 + table.shape[1]], starts.long(), lens.long())):
        got, lse = capi.page_attention(q, cache, scales, t, s + 7, l, b.scale, return_lse=True, **rule)
        _close(got[7:40], lse[7:40], want, torch.bfloat16, 128)
        for part in (slice(0, 7), slice(40, None)):
            assert bool((got[part] == 0).all()) and bool(lse[part].isneginf().all())


@pytest.mark.parametrize("bits, seen", RULES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_more_requests_than_threads(capi, bits, seen, dim):
    rng = np.random.default_rng(dim)
    lens = rng.integers(0, 24, 600)
    q = np.minimum(rng.integers(0, 9, 600), lens)
    b = Batch(dim, lens, q, 2, 1, dim, 16, torch.bfloat16, bits, seen)
    for hint in (9, 1000):
        _check(capi, b, max_query_len=hint)
    if seen == "tree":
        _check(capi, b, max_query_len=1000, window=3, sinks=1)


@pytest.mark.parametrize("bits, seen", RULES)
@pytest.mark.parametrize("q", [5, 150])
def test_a_graph_and_another_stream(capi, bits, seen, q):
    b = Batch(12, [900, 240, 300], [q, q, q], 8, 2, 128, 16, torch.bfloat16, bits, seen)
    args, rule = b.args(), b.rule(capi)
    plain = capi.page_attention(*args, b.scale, max_query_len=q, **rule)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late = args[0] + 0
        got = capi.page_attention(late, *args[1:], b.scale, max_query_len=q, **rule)
    side.synchronize()
    assert torch.equal(got, plain)
    parents = torch.as_tensor(b.parents).int().to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        if seen == "tree":
            rule = dict(tree=capi.page_tree(parents, args[4], args[5])[0])
        kept = capi.page_attention(*args, b.scale, max_query_len=q, **rule)
    for i in range(4):
        args[0].normal_()
        args[5].copy_(torch.tensor([900 - 100 * i, 240 - i, 217 + i], dtype=torch.int32))
        if seen == "tree":
            parents.copy_(torch.as_tensor(np.concatenate([grown(b.rng, q, KINDS[(i + k) % 5]) for k in range(3)])))
            rule = dict(tree=capi.page_tree(parents, args[4], args[5])[0])
        want = capi.page_attention(*args, b.scale, max_query_len=q, **rule)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, want)


@pytest.mark.parametrize("q", [1, 50])
def test_offsets_beyond_32_bits(capi, q):
    """Pages more than 4 GiB apart, 8 bits."""
    b = Batch(9, [300], [q], 4, 1, 128, 16, torch.bfloat16, 8)
    query, cache, scales, table, starts, lens = b.args()
    far = (1 << 32) // len(cache) // 16 * 16 * 2
    room = torch.zeros(far * len(cache), dtype=torch.uint8, device=DEV)
    apart = room.as_strided(cache.shape, (far, *cache.stride()[1:]))
    apart.copy_(cache.view(torch.uint8))
    _close(capi.page_attention(query, apart.view(torch.float8_e4m3fn), scales, table, starts, lens, b.scale), None, b.want(),
           torch.bfloat16, 128)


def test_refusals(capi):
    b = Batch(1, [20, 30], [1, 2], 4, 2, 64, 16, torch.bfloat16, 4, "tree")
    args, tree = b.args(), b.rule(capi)["tree"]
    for text, kw in (("does not go with causal", dict(tree=tree, causal=False)), ("no window", dict(causal=False, window=5)),
                     ("page_tree makes", dict(tree=tree[:2])), ("page_tree makes", dict(tree=tree.long())),
                     ("page_tree makes", dict(tree=tree[:, :3])), ("CUDA", dict(tree=tree.cpu()))):
        with pytest.raises(RuntimeError, match=text):
            capi.page_attention(*args, **kw)
    with pytest.raises(RuntimeError, match="requires a gradient"):
        capi.page_attention(args[0].clone().requires_grad_(), *args[1:], tree=tree)
    odd = torch.zeros(13, dtype=torch.int32, device=DEV)[1:].view(3, 4)  # does not begin on 16 bytes
    odd.copy_(tree)
    assert torch.equal(capi.page_attention(*args, tree=odd), capi.page_attention(*args, tree=tree))
