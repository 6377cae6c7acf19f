"""The paged 4-bit cache on the GPU against its definition in 64 bits (oracle/paged.py). Plans, codes and scale bytes
are whole numbers and have to be equal; what rows stand for is exact in float32 and bfloat16."""
import numpy as np
import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _empty(pages, heads, page, dim, fill=0xA5):
    return (torch.full((pages, heads, 2, page, dim // 2), fill, dtype=torch.uint8, device=DEV),
            torch.full((pages, heads, 2, dim // 32, page), fill, dtype=torch.uint8, device=DEV))


def _rows(gen, shape, dtype):
    """Rows of all magnitudes: blocks of very different size, zeros of both signs, ties, values at the edge of a step."""
    x = torch.randn(shape, generator=gen, dtype=torch.float64)
    n = x.numel() // 32
    b = x.view(n, 32)
    most = 14 if dtype == torch.float16 else 120
    b *= torch.exp2(torch.randint(-most, most, (n, 1), generator=gen).double())
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 6.96875, -0.0, 0.0, -0.25, -7.0, 1.0, 3.0])
    for i in range(0, n, 5):
        b[i] = ties[torch.randint(0, 16, (32,), generator=gen)] * 2.0 ** int(torch.randint(-10, 10, (1,), generator=gen))
    b[1 % n] = 0
    b[2 % n] = -0.0
    b[3 % n] *= 2.0 ** -130 / b[3 % n].abs().max()                   # below the smallest normal number
    return x.to(dtype)


def _np(t):
    return t.double().cpu().numpy()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tokens, heads, page, wide", [(1, 1, 16, 8), (37, 3, 32, 4), (300, 8, 64, 8), (129, 2, 256, 4),
                                                       (1000, 1, 128, 8)])
def test_rows_go_in_and_come_out(capi, dtype, dim, tokens, heads, page, wide):
    gen = torch.Generator().manual_seed(tokens * dim)
    joint = _rows(gen, (tokens, 3 * heads, dim), dtype).to(DEV)       # strides of a joint projection
    keys, values = joint[:, heads:2 * heads], joint[:, 2 * heads:]
    pages = -(-tokens // page) + 2
    cache, scales = _empty(pages, heads, page, dim)
    slots = torch.randperm(pages * page, generator=gen)[:tokens].to(torch.int64 if wide == 8 else torch.int32)
    slots[::7] = -1
    if tokens > 20:
        slots[3], slots[11] = pages * page, 2**31 - 1                 # outside the cache as well
    want_cache, want_scales = cache.cpu().numpy(), scales.cpu().numpy()
    paged.rows_set(want_cache, want_scales, slots.tolist(), _np(keys), _np(values))
    capi.page_set(cache, scales, slots.to(DEV), keys, values)
    assert np.array_equal(scales.cpu().numpy(), want_scales)
    assert np.array_equal(cache.cpu().numpy(), want_cache)            # places that no slot names keep what they held
    back = slots[torch.randperm(tokens, generator=gen)]
    want = paged.rows_fetch(want_cache, want_scales, back.tolist())
    for out_type in (torch.float32, torch.bfloat16, torch.float16):
        got = capi.page_fetch(cache, scales, back.to(DEV), out_type)
        for g, w in zip(got, want):
            w = torch.from_numpy(w).float().to(out_type)
            assert g.dtype == out_type and g.is_contiguous()
            assert torch.equal(g.cpu().double().nan_to_num(nan=1e300), w.double().nan_to_num(nan=1e300))


def test_infinities_and_nan_mark_their_block_only(capi):
    cache, scales = _empty(2, 1, 16, 64)
    x = torch.ones((4, 1, 64), dtype=torch.bfloat16, device=DEV)
    x[0, 0, 5], x[1, 0, 40], x[2, 0, 0] = float("nan"), float("inf"), -float("inf")
    slots = torch.tensor([0, 17, 31, 8], device=DEV)
    capi.page_set(cache, scales, slots, x, torch.ones_like(x))
    keys, values = capi.page_fetch(cache, scales, slots, torch.float32)
    bad = torch.zeros((4, 64), dtype=torch.bool, device=DEV)
    bad[0, :32] = bad[1, 32:] = bad[2, :32] = True
    assert torch.equal(keys[:, 0].isnan(), bad) and bool((keys[:, 0][~bad] == 1).all()) and bool((values == 1).all())


@pytest.mark.parametrize("offset", [0, 1])
def test_rows_of_any_alignment_and_pages_that_lie_apart(capi, offset):
    gen = torch.Generator().manual_seed(3)
    flat = _rows(gen, (40 * 5 * 128 + 32,), torch.bfloat16).to(DEV)[offset:]
    keys = flat[:40 * 5 * 128].view(40, 5, 128)[:, 1:3]
    values = flat[:40 * 5 * 128].view(5, 40, 128).transpose(0, 1)[:, 2:4]
    both = torch.full((2, 6, 2, 2, 16, 64), 7, dtype=torch.uint8, device=DEV)    # two layers' pages side by side
    bs = torch.full((6, 2, 2, 2, 4, 16), 9, dtype=torch.uint8, device=DEV)
    cache, scales = both[1], bs[:, 1]
    slots = torch.randperm(96, generator=gen)[:40].to(DEV)
    want_cache, want_scales = cache.cpu().numpy().copy(), scales.cpu().numpy().copy()
    paged.rows_set(want_cache, want_scales, slots.tolist(), _np(keys), _np(values))
    capi.page_set(cache, scales, slots, keys, values)
    assert np.array_equal(cache.cpu().numpy(), want_cache) and np.array_equal(scales.cpu().numpy(), want_scales)
    assert bool((both[0] == 7).all()) and bool((bs[:, 0] == 9).all())
    got = capi.page_fetch(cache, scales, slots, torch.float32)
    for g, w in zip(got, paged.rows_fetch(want_cache, want_scales, slots.tolist())):
        assert np.array_equal(_np(g), w)


def test_no_rows(capi):
    cache, scales = _empty(2, 4, 16, 128)
    none = torch.empty((0,), dtype=torch.int64, device=DEV)
    x = torch.empty((0, 4, 128), dtype=torch.float16, device=DEV)
    capi.page_set(cache, scales, none, x, x)
    assert [t.shape for t in capi.page_fetch(cache, scales, none, torch.float16)] == [(0, 4, 128)] * 2
    got = capi.page_fetch(cache[:0], scales[:0], torch.tensor([0, -1], device=DEV), torch.float16)
    assert bool((got[0] == 0).all())


PLANS = [
    # requests, longest cached, most new, page, room in the table, free pages (share of what is needed), room for tokens
    (1, 0, 1, 16, 1.0, 1.0, 1.0), (1, 1000, 700, 32, 1.0, 1.0, 1.0), (7, 40, 1, 16, 1.0, 1.0, 1.3),
    (64, 300, 40, 16, 1.0, 1.0, 1.0), (64, 300, 40, 64, 0.5, 1.0, 1.0), (64, 300, 40, 16, 1.0, 0.3, 1.0),
    (200, 100, 90, 16, 1.0, 0.0, 0.4), (255, 17, 2, 16, 1.0, 1.0, 1.0), (256, 17, 2, 16, 1.0, 1.0, 1.0),
    (257, 17, 2, 128, 1.0, 1.0, 2.0), (1025, 50, 9, 16, 1.0, 0.9, 1.0), (5000, 33, 3, 16, 1.0, 1.0, 1.0),
    (20000, 20, 2, 16, 1.0, 1.0, 1.1), (3, 9, 30000, 256, 1.0, 1.0, 1.0), (100, 4000, 0, 16, 1.0, 1.0, 1.0),
]


@pytest.mark.parametrize("case", PLANS, ids=[str(c[:4]) for c in PLANS])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_plan(capi, case, dtype):
    n, longest, most, page, room, supply, space = case
    rng = np.random.default_rng(n + longest)
    cached, new = rng.integers(0, longest + 1, n), rng.integers(0, most + 1, n)
    cached[rng.random(n) < 0.2] = 0
    new[rng.random(n) < 0.2] = 0
    if n > 5:
        cached[2], new[4] = -3, -1                                    # count as 0
    have, end = -(-np.maximum(cached, 0) // page), -(-(np.maximum(cached, 0) + np.maximum(new, 0)) // page)
    width = max(1, int(end.max() * room))
    needed = int((end - have).sum())
    tokens = int(np.maximum(new, 0).sum() * space)
    pool = rng.permutation(int(end.sum()) + 9).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    at = 0
    for b in range(n):
        w = min(have[b], width)
        table[b, :w] = pool[at:at + w]
        at += w
    free = rng.permutation(1 << 20)[:int(needed * supply)].astype(np.int32)
    wide = torch.full((n, width + 3), -5, dtype=torch.int32, device=DEV)
    wide[:, 1:width + 1] = torch.from_numpy(table).to(DEV)
    dev_table = wide[:, 1:width + 1]                                  # rows lie apart
    want = paged.plan(cached, new, table, free, page, tokens)
    got = capi.page_plan(torch.from_numpy(cached).to(DEV, dtype), torch.from_numpy(new).to(DEV, dtype), dev_table,
                         torch.from_numpy(free).to(DEV), page, tokens)
    for name, g, w in zip(("query_starts", "kv_lens", "positions", "slots", "counts"), got, want):
        assert np.array_equal(g.cpu().numpy(), w), name
    assert [g.dtype for g in got] == [torch.int32] * 3 + [torch.int64] * 2
    assert np.array_equal(dev_table.cpu().numpy(), table)
    assert bool((wide[:, 0] == -5).all()) and bool((wide[:, width + 1:] == -5).all())


def test_plan_of_nothing(capi):
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)
    got = capi.page_plan(i(0), i(0), i(0, 4), i(0), 16, 3)
    assert got[0].tolist() == [0] and got[2].tolist() == [-1] * 3 and got[3].tolist() == [-1] * 3 and got[4].tolist() == [0, 0]
    got = capi.page_plan(i(2), i(2) + 1, i(2, 0), i(5), 16, 2)        # a table without room
    assert got[3].tolist() == [-1, -1] and got[4].tolist() == [2, 2]
    got = capi.page_plan(i(2), i(2) + 1, i(2, 1), i(5), 16, 0)        # no room for tokens
    assert got[2].numel() == 0 and got[4].tolist() == [2, 2]


def test_operators_on_another_stream(capi):
    """plan, set and fetch queued on a stream of the caller's, behind work that makes their inputs."""
    gen = torch.Generator().manual_seed(0)
    x = _rows(gen, (64, 2, 128), torch.bfloat16).to(DEV)
    cache, scales = _empty(8, 2, 16, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        y = x + 0
        lens = torch.full((4,), 16, dtype=torch.int32, device=DEV)
        table = torch.full((4, 2), -1, dtype=torch.int32, device=DEV)
        _, _, _, slots, _ = capi.page_plan(lens - 16, lens, table, torch.arange(8, dtype=torch.int32, device=DEV), 16, 64)
        capi.page_set(cache, scales, slots, y, y)
        k, v = capi.page_fetch(cache, scales, slots, torch.float32)
    side.synchronize()
    code, byte = paged.encode(_np(x))
    assert slots.tolist() == list(range(64))
    assert np.array_equal(_np(k), paged.decode(code, byte)) and torch.equal(k, v)


def test_refusals(capi):
    cache, scales = _empty(4, 2, 16, 128)
    x = torch.zeros((3, 2, 128), dtype=torch.bfloat16, device=DEV)
    s = torch.zeros(3, dtype=torch.int64, device=DEV)
    def no(text, f, *args, **kw):
        with pytest.raises((RuntimeError, ValueError), match=text):
            f(*args, **kw)
    no("CUDA tensor", capi.page_set, cache.cpu(), scales, s, x, x)
    no("CUDA tensor", capi.page_set, cache, scales, s.cpu(), x, x)
    no("CUDA tensor", capi.page_set, cache, scales, s, x.cpu(), x)
    no("uint8", capi.page_set, cache.int(), scales, s, x, x)
    no("scales must be", capi.page_set, cache, scales[:, :1], s, x, x)
    no("cache must be", capi.page_set, cache[:, :, 0], scales, s, x, x)
    no("contiguous", capi.page_set, cache.transpose(3, 4).contiguous().transpose(3, 4), scales, s, x, x)
    no("int32 or int64", capi.page_set, cache, scales, s.float(), x, x)
    no("keys and values must be", capi.page_set, cache, scales, s, x[:2], x)
    no("one type", capi.page_set, cache, scales, s, x, x.float())
    no("float32, float16 or bfloat16", capi.page_set, cache, scales, s, x.double(), x.double())
    no("float32, float16 or bfloat16", capi.page_fetch, cache, scales, s, torch.int8)
    no("64, 128 or 256", capi.page_fetch, *_empty(2, 1, 16, 32), s, torch.float32)
    no("a page must hold", capi.page_fetch, *_empty(2, 1, 24, 64), s, torch.float32)
    i = torch.zeros(3, dtype=torch.int32, device=DEV)
    t = torch.zeros((3, 2), dtype=torch.int32, device=DEV)
    no("int32 tensor", capi.page_plan, i, i, t.long(), i, 16, 4)
    no("one type", capi.page_plan, i, i.long(), t, i, 16, 4)
    no("int32 or int64", capi.page_plan, i.float(), i, t, i, 16, 4)
    no("a length for each", capi.page_plan, i[:2], i, t, i, 16, 4)
    no("free_pages", capi.page_plan, i, i, t, i.long(), 16, 4)
    no("max_tokens", capi.page_plan, i, i, t, i, 16, -1)
    no("a page must hold", capi.page_plan, i, i, t, i, 20, 4)
    no("contiguous", capi.page_plan, i, i, torch.zeros((2, 3), dtype=torch.int32, device=DEV).t(), i, 16, 4)
    no("overlap", capi.page_plan, i, i, t[:1].expand(3, 2), i, 16, 4)


@pytest.mark.parametrize("room", [1.0, 0.9, 1.2])
def test_plan_of_long_prompts(capi, room):
    """Hundreds of thousands of tokens: four in a row to a thread, across the ends of requests and pages."""
    rng = np.random.default_rng(5)
    cached, new = rng.integers(0, 100, 50), rng.integers(0, 9000, 50)
    new[3], new[4], new[5], new[20] = 1, 0, 2, 0
    end = -(-(cached + new) // 16)
    table = np.full((50, int(end.max()) - 3), -1, np.int32)                # the longest requests outgrow it
    table[:, :7] = rng.permutation(1 << 20)[:350].reshape(50, 7)
    free = rng.permutation(1 << 20)[:int((end - -(-cached // 16)).sum()) - 9].astype(np.int32)
    tokens = int(new.sum() * room) | 1
    dev_table = torch.from_numpy(table.copy()).to(DEV)
    want = paged.plan(cached, new, table, free, 16, tokens)
    got = capi.page_plan(torch.from_numpy(cached).to(DEV), torch.from_numpy(new).to(DEV), dev_table,
                         torch.from_numpy(free).to(DEV), 16, tokens)
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), w)
    assert np.array_equal(dev_table.cpu().numpy(), table)
