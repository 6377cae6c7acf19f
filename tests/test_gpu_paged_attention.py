"""Attention over the paged 4-bit cache against its definition in 64 bits (oracle/paged.py).

Bounds, per row, head and dimension, from the definition alone. With u the unit round-off of the type (2^-9 for
bfloat16, 2^-12 for float16), A = sum_j w_j |V_j| and S the largest scale * sum_d |q_d K_jd| of the row:
  out: one rounding of the result, u |out|, and below float16's smallest normal number half of its spacing there, 2^-25;
  weights below the smallest normal number of 32 bits, 2^-126 each, which may be lost: 2^-100 for all tokens; the weights rounded to no fewer than the type's bits before they meet V,
  u A; scores summed in 32 bits, each off by at most (dim + 8) 2^-24 S, which moves a weight and the normaliser by that
  part each; exp, sums and joins in 32 bits, 2^-16 A together. Twice the sum is allowed.
  lse: (dim + 8) 2^-24 S + 2^-16 + 2^-22 |lse|, twice.
"""
import numpy as np
import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROUND = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -12}
TINY = {torch.bfloat16: 2.0 ** -100, torch.float16: 2.0 ** -25}


class Batch:
    """Requests in a cache whose other places hold garbage: pages of no request, places behind a request's end."""

    def __init__(self, seed, kv_lens, query_lens, heads, kv_heads, dim, page, dtype, spread=1.5, width=None):
        gen = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        kv_lens, query_lens = np.asarray(kv_lens), np.asarray(query_lens)
        count = -(-kv_lens // page)
        pages = int(count.sum()) + 3
        order = rng.permutation(pages)
        self.cache = torch.randint(0, 256, (pages, kv_heads, 2, page, dim // 2), generator=gen, dtype=torch.uint8)
        self.scales = torch.full((pages, kv_heads, 2, dim // 32, page), 255, dtype=torch.uint8)
        width = max(1, int(count.max())) if width is None else width
        self.table = torch.full((len(kv_lens), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(count):
            mine = order[at:at + n]
            at += n
            self.table[b, :min(n, width)] = torch.from_numpy(mine[:width]).int()
            for i, p in enumerate(mine):
                live = min(page, int(kv_lens[b]) - i * page)
                self.scales[p, ..., :live] = torch.randint(124, 128, (kv_heads, 2, dim // 32, live), generator=gen).byte()
        self.starts = torch.tensor(np.concatenate([[0], np.cumsum(query_lens)]), dtype=torch.int32)
        self.kv_lens = torch.tensor(kv_lens, dtype=torch.int32)
        self.query = (torch.randn((int(self.starts[-1]), heads, dim), generator=gen) * spread).to(dtype)
        self.scale = dim ** -0.5

    def args(self):
        return [t.to(DEV) for t in (self.query, self.cache, self.scales, self.table, self.starts, self.kv_lens)]

    def want(self, **kw):
        return paged.attention(self.query.double().numpy(), self.cache.numpy(), self.scales.numpy(), self.table.numpy(),
                               self.starts.numpy(), self.kv_lens.numpy(), self.scale, **kw)


def _close(got, lse, want, dtype, dim):
    out, wlse, spread, top = want
    u = ROUND[dtype]
    score = ((dim + 8) * 2.0 ** -24 * top)[..., None]
    bound = 2 * (u * np.abs(out) + TINY[dtype] + (u + 2 * score + 2.0 ** -16) * spread)
    g = got.double().cpu().numpy()
    assert g.shape == out.shape and got.dtype == dtype and got.is_contiguous()
    assert np.array_equal(np.isnan(g), np.isnan(out))
    far = np.nan_to_num(np.abs(g - out) - bound, nan=0.0)
    assert far.max(initial=-1) <= 0, "out is off by %.3g over its bound at %s" % (far.max(), np.unravel_index(far.argmax(), far.shape))
    if lse is not None:
        l = lse.double().cpu().numpy()
        assert lse.dtype == torch.float32 and np.array_equal(np.isneginf(l), np.isneginf(wlse))
        fine = np.isfinite(wlse)
        assert np.array_equal(np.isnan(l), np.isnan(wlse))
        assert (np.abs(l[fine] - wlse[fine]) <= 2 * (score[..., 0] + 2.0 ** -16 + 2.0 ** -22 * np.abs(wlse))[fine]).all()


def _check(capi, batch, **kw):
    query = batch.query
    hint = kw.pop("max_query_len", int(batch.starts.diff().max()) if len(batch.kv_lens) else 0)
    got, lse = capi.page_attention(*batch.args(), batch.scale, max_query_len=hint, return_lse=True, **kw)
    _close(got, lse, batch.want(**kw), query.dtype, query.shape[2])
    return got, lse


HEADS = [(1, 1), (4, 1), (6, 2), (5, 5), (8, 1), (14, 2), (16, 1), (24, 1), (40, 1), (8, 4)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads, kv_heads", HEADS)
def test_single_tokens(capi, dtype, dim, heads, kv_heads):
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 128, 129, 300, 0, 257]
    q = [1] * len(lens)
    q[13] = 1                                                          # a query with nothing to look at
    _check(capi, Batch(heads * dim, lens, q, heads, kv_heads, dim, 16, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads, kv_heads", [(4, 2), (10, 2), (3, 1)])
def test_several_tokens(capi, dtype, dim, page, heads, kv_heads):
    """Whole prompts, chunks behind a cached part, requests without new tokens."""
    lens, q = [1, 40, 77, 160, 9, 130, 300, 33], [1, 40, 5, 31, 0, 130, 2, 17]
    _check(capi, Batch(page + dim, lens, q, heads, kv_heads, dim, page, dtype))


@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (7, 3), (16, 16), (33, 4), (64, 0), (100, 50), (128, 1),
                                           (200, 300), (100000, 5)])
@pytest.mark.parametrize("dtype, dim, page, heads, kv_heads", [
    (torch.bfloat16, 128, 16, 8, 2), (torch.float16, 64, 32, 3, 1), (torch.bfloat16, 256, 64, 2, 2)])
def test_windows_and_sinks(capi, window, sinks, dtype, dim, page, heads, kv_heads):
    lens, q = [1, 400, 77, 260, 500, 34, 150], [1, 1, 77, 50, 3, 0, 129]
    _check(capi, Batch(window + dim, lens, q, heads, kv_heads, dim, page, dtype), window=window, sinks=sinks)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q", [1, 6, 90])
def test_windows_over_pages_that_were_given_back(capi, dim, q):
    b = Batch(dim, [600, 333, 700], [q, q, q], 8, 2, dim, 16, torch.bfloat16)
    kept = {k: b.want(window=120, sinks=9)[k] for k in (0,)}
    for r, n in enumerate([600, 333, 700]):
        first = (n - q - 120 + 1) // 16
        gone = b.table[r, 1:first].clone()
        b.table[r, 1:first] = -1
        b.scales[gone.long()] = 255                                    # what they hold now is another request's business
    got, _ = _check(capi, b, window=120, sinks=9)
    assert np.array_equal(b.want(window=120, sinks=9)[0], kept[0])


def test_pages_that_are_missing_are_not_seen(capi):
    for dim, q in ((128, 1), (64, 3), (256, 70), (128, 200)):
        b = Batch(dim + q, [500, 260, 300], [q, q, q], 4, 2, dim, 32, torch.bfloat16)
        b.table[0, 2:5] = -1
        b.table[1, :] = -1                                             # a request that sees nothing
        b.table[2, 0], b.table[2, 3] = len(b.cache), 2**31 - 1         # no pages of this cache
        _check(capi, b)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_more_queries_than_tokens(capi, dim):
    """Rows in front of the request's first token see nothing; a table may be shorter than kv_lens says."""
    b = Batch(5, [3, 0, 50], [9, 4, 60], 4, 1, dim, 16, torch.float16)
    got, lse = _check(capi, b)
    assert bool((got[:6] == 0).all()) and bool((got[9:13] == 0).all()) and bool(lse[9:13].isneginf().all())
    b = Batch(6, [200, 90], [1, 20], 4, 1, dim, 16, torch.float16, width=3)
    _check(capi, b)


def test_rows_of_no_request(capi):
    b = Batch(7, [50, 60, 70], [1, 30, 2], 4, 2, 128, 16, torch.bfloat16)
    want = list(b.want())
    query, cache, scales, table, starts, lens = b.args()
    padded = torch.cat([query[:7], query, query[:90]])                 # rows in front and behind
    got, lse = capi.page_attention(padded, cache, scales, table, starts + 7, lens, b.scale, return_lse=True)
    _close(got[7:40], lse[7:40], want, torch.bfloat16, 128)
    for part in (slice(0, 7), slice(40, None)):
        assert bool((got[part] == 0).all()) and bool(lse[part].isneginf().all())
    got = capi.page_attention(padded, cache, scales, table[:0], starts[:1], lens[:0], b.scale)
    assert bool((got == 0).all())


@pytest.mark.parametrize("hint", [0, 1, 2, 17, 64, 1000])
@pytest.mark.parametrize("dim, heads, kv_heads", [(128, 8, 2), (64, 20, 1), (256, 4, 2)])
def test_the_hint_only_chooses_the_kernel(capi, hint, dim, heads, kv_heads):
    b = Batch(hint, [400, 33, 90, 150], [1, 33, 2, 64], heads, kv_heads, dim, 16, torch.bfloat16)
    _check(capi, b, max_query_len=hint)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_work_split_over_long_requests(capi, dtype):
    """Few rows and many tokens: parts are computed apart and joined; beside them short requests."""
    _check(capi, Batch(1, [9001], [1], 5, 1, 128, 32, dtype))
    _check(capi, Batch(2, [5, 6000, 1, 3000, 17], [1, 2, 1, 1, 3], 4, 2, 64, 16, dtype))
    _check(capi, Batch(3, [4100], [20], 8, 1, 256, 64, dtype))
    _check(capi, Batch(4, [5000, 3], [40, 3], 4, 1, 128, 16, dtype), window=2500, sinks=70)


@pytest.mark.parametrize("q", [1, 4, 100])
def test_not_a_number_where_it_is_seen_and_nowhere_else(capi, q):
    for dim in (64, 128, 256):
        b = Batch(dim, [200, 150], [q, q], 4, 2, dim, 16, torch.bfloat16)
        at = lambda r, j: int(b.table[r, j // 16])
        b.scales[at(0, 130), 0, 1, 1, 130 % 16] = 255                  # one block of one value of head 0
        b.scales[at(0, 120), 0, 1, 0, 120 % 16] = 255
        b.scales[at(1, 149), 1, 0, 0, 149 % 16] = 255                  # a key that only the last row sees
        want = b.want(window=70)
        assert np.isnan(want[0]).any() and not np.isnan(want[0]).all()
        _check(capi, b, window=70)


def test_infinite_queries_and_extreme_scores(capi):
    b = Batch(1, [90, 100], [1, 40], 4, 2, 128, 16, torch.bfloat16, spread=1.0)
    b.query[0] *= 2.0 ** 10                                            # one token takes all the weight
    b.query[5] = 0                                                     # equal weights
    _check(capi, b)
    b.query[3, 1, 7] = float("nan")
    got = capi.page_attention(*b.args(), b.scale)
    assert bool(got[3, 1].isnan().all()) and not bool(got[:3].isnan().any()) and not bool(got[4:].isnan().any())
    assert not bool(got[3, [0, 2, 3]].isnan().any())
    b = Batch(2, [90, 100], [1, 40], 4, 2, 128, 16, torch.float16)
    big = b.scales != 255
    b.scales[:, :, 0][big[:, :, 0]] += 60                              # scores far outside of what exp takes
    b.scale = 2.0 ** -60 * 128 ** -0.5
    _check(capi, b)
    b.scale = 0.0
    _check(capi, b)
    b.scale = -0.05 * 2.0 ** -60
    _check(capi, b)


def test_strides_and_widths(capi):
    b = Batch(4, [100, 200, 30], [3, 40, 1], 6, 2, 128, 16, torch.bfloat16)
    want = b.want()
    query, cache, scales, table, starts, lens = b.args()
    joint = torch.randn((44, 10, 128), device=DEV).bfloat16()
    joint[:, 2:8] = query
    wide = torch.full((3, 40), 1, dtype=torch.int32, device=DEV)
    wide[:, 4:4 + table.shape[1]] = table
    odd = torch.empty(query.numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].view(query.shape)
    odd.copy_(query)
    turned = query.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    layers = torch.zeros((len(cache), 3, *cache.shape[1:]), dtype=torch.uint8, device=DEV)
    layers[:, 1] = cache
    for q, c, s, t, i, l in ((joint[:, 2:8], cache, scales, wide[:, 4:4 + table.shape[1]], starts.long(), lens.long()),
                             (odd, layers[:, 1], scales, table, starts, lens), (turned, cache, scales, table, starts, lens)):
        got, lse = capi.page_attention(q, c, s, t, i, l, b.scale, return_lse=True)
        _close(got, lse, want, torch.bfloat16, 128)
    assert torch.equal(capi.page_attention(query, cache, scales, table, starts, lens),
                       capi.page_attention(query, cache, scales, table, starts, lens, 128 ** -0.5))


@pytest.mark.parametrize("q", [1, 50])
def test_offsets_beyond_32_bits(capi, q):
    """Pages more than 4 GiB apart."""
    b = Batch(9, [300], [q], 4, 1, 128, 16, torch.bfloat16)
    want = b.want()
    query, cache, scales, table, starts, lens = b.args()
    far = (1 << 32) // len(cache) // 16 * 16 * 2
    room = torch.zeros(far * len(cache), dtype=torch.uint8, device=DEV)
    apart = room.as_strided(cache.shape, (far, *cache.stride()[1:]))
    apart.copy_(cache)
    got = capi.page_attention(query, apart, scales, table, starts, lens, b.scale)
    _close(got, None, want, torch.bfloat16, 128)
    x = torch.ones((1, 1, 128), device=DEV)
    slot = torch.tensor([len(cache) * 16 - 1], device=DEV)
    capi.page_set(apart, scales, slot, x, 2 * x)
    k, v = capi.page_fetch(apart, scales, slot, torch.float32)
    assert bool((k == 1).all()) and bool((v == 2).all())


def test_the_same_call_gives_the_same_bits(capi):
    for lens, q in (([9001, 40], [1, 1]), ([3000, 900], [64, 300])):
        b = Batch(11, lens, q, 8, 2, 128, 16, torch.bfloat16)
        args = b.args()
        first = capi.page_attention(*args, b.scale)
        for _ in range(5):
            assert torch.equal(capi.page_attention(*args, b.scale), first)


def test_another_stream_and_a_graph(capi):
    b = Batch(12, [900, 40, 300], [1, 1, 1], 8, 2, 128, 16, torch.bfloat16)
    args = b.args()
    plain = capi.page_attention(*args, b.scale, max_query_len=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late = args[0] + 0
        got = capi.page_attention(late, *args[1:], b.scale, max_query_len=1)
    side.synchronize()
    assert torch.equal(got, plain)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = capi.page_attention(*args, b.scale, max_query_len=1)
    for i in range(4):
        args[0].normal_()
        args[5].copy_(torch.tensor([900 - 100 * i, 40 - i, 17 + i], dtype=torch.int32))
        want = capi.page_attention(*args, b.scale, max_query_len=1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, want)


def test_a_step_as_a_program_makes_it(capi):
    """Plan, rows in, attention: the prompt at once, and token by token, give what the definition gives."""
    gen = torch.Generator().manual_seed(0)
    page, heads, kv_heads, dim = 16, 4, 2, 64
    cache = torch.full((9, kv_heads, 2, page, dim // 2), 255, dtype=torch.uint8, device=DEV)
    scales = torch.full((9, kv_heads, 2, dim // 32, page), 255, dtype=torch.uint8, device=DEV)
    table = torch.full((2, 5), -1, dtype=torch.int32, device=DEV)
    free = torch.tensor([7, 0, 3, 8, 1, 2, 6], dtype=torch.int32, device=DEV)
    cached = torch.zeros(2, dtype=torch.int32, device=DEV)
    taken = 0
    for new in ([33, 15], [1, 1], [1, 1], [4, 0]):
        new = torch.tensor(new, dtype=torch.int32, device=DEV)
        n = int(new.sum())
        q, k, v = (torch.randn((n, h, dim), generator=gen).bfloat16().to(DEV) for h in (heads, kv_heads, kv_heads))
        starts, lens, pos, slots, counts = capi.page_plan(cached, new, table, free[taken:], page, n)
        taken += int(counts[1])
        capi.page_set(cache, scales, slots, k, v)
        got = capi.page_attention(q, cache, scales, table, starts, lens)
        want = paged.attention(q.double().cpu().numpy(), cache.cpu().numpy(), scales.cpu().numpy(), table.cpu().numpy(),
                               starts.cpu().numpy(), lens.cpu().numpy(), dim ** -0.5)
        assert np.isfinite(want[0]).all()
        _close(got, None, want, torch.bfloat16, dim)
        cached = lens


def test_refusals(capi):
    b = Batch(1, [20, 30], [1, 2], 4, 2, 64, 16, torch.bfloat16)
    good = b.args()
    def no(text, at=None, value=None, **kw):
        args = list(good)
        if at is not None:
            args[at] = value
        with pytest.raises((RuntimeError, ValueError), match=text):
            capi.page_attention(*args, **kw)
    query, cache, scales, table, starts, lens = good
    no("float16 or bfloat16", 0, query.float())
    no("must be \\[tokens", 0, query[..., :32])
    no("evenly", 0, query[:, :3])
    no("CUDA tensor", 0, query.cpu())
    no("uint8", 1, cache.int())
    no("scales must be", 2, scales[..., :8])
    no("int32 tensor", 3, table.long())
    no("CUDA tensor", 3, table.cpu())
    no("one entry more", 4, starts[:-1])
    no("one entry more", 5, lens[:1])
    no("one type", 5, lens.long())
    no("int32 or int64", 4, starts.float())
    no(">= 0", window=-1)
    no(">= 0", sinks=-2)
    no(">= 0", max_query_len=-1)
    no("finite", softmax_scale=float("inf"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_rows(capi, dtype, dim):
    """Requests of hundreds of rows: not a number in some rows' sight, one token that takes all weight, parts to join."""
    b = Batch(dim + 1, [700, 300, 5], [290, 300, 5], 6, 2, dim, 16, dtype)
    at = lambda r, j: int(b.table[r, j // 16])
    b.scales[at(0, 520), 0, 1, 1, 520 % 16] = 255                      # a value's block that the later rows see
    b.scales[at(0, 690), 1, 0, 0, 690 % 16] = 255                      # a key that the last rows see
    b.scales[at(1, 3), 1, 1, 0, 3] = 250 if dtype == torch.bfloat16 else 140   # values near the end of the type's range
    b.query[7] *= 2.0 ** 9
    b.query[400, 1] *= -2.0 ** 9
    want = b.want()
    assert np.isnan(want[0]).any() and not np.isnan(want[0]).all()
    _check(capi, b)
    _check(capi, b, window=130, sinks=20)
    _check(capi, Batch(3, [2300, 40], [280, 1], 2, 1, dim, 32, dtype))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_more_requests_than_threads(capi, dim):
    rng = np.random.default_rng(dim)
    lens = rng.integers(0, 24, 600)
    q = np.minimum(rng.integers(0, 5, 600), lens)
    b = Batch(dim, lens, q, 2, 1, dim, 16, torch.bfloat16)
    for hint in (4, 1000):                                             # the kernels for few rows and for many
        _check(capi, b, max_query_len=hint)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window, sinks", [(0, 0), (1, 1), (7, 3), (64, 0), (100, 50), (200, 300)])
def test_ragged_requests_in_the_kernel_for_many_rows(capi, dtype, dim, window, sinks):
    """A hint that is too great: single tokens, chunks and prompts as items of many rows; pages missing or given back; values
    that are not a number where some rows, all or none see them."""
    b = Batch(dim + window, [1, 400, 77, 260, 500, 34, 150], [1, 1, 77, 50, 3, 0, 129], 9, 3, dim, 32, dtype)
    _check(capi, b, window=window, sinks=sinks, max_query_len=4000)
    at = lambda r, j: int(b.table[r, j // 32])
    b.scales[at(6, 75), 1, 1, 0, 75 % 32] = 255                        # a value that later rows see, and windows pass
    b.scales[at(3, 2), 0, 1, 1, 2] = 255
    b.scales[at(2, 40), 2, 0, 1, 40 % 32] = 255                        # a key
    b.table[1, 2:5] = -1
    b.table[4, 0], b.table[4, 9] = len(b.cache), 2**31 - 1
    b.table[5, :] = -1
    _check(capi, b, window=window, sinks=sinks, max_query_len=4000)
