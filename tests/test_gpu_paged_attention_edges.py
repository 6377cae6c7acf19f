"""Attention over the paged 4-bit cache at the edges of its calls."""
import ctypes

import numpy as np
import pytest
import torch

from test_gpu_paged_attention import Batch, _check

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("tokens, heads, kv_heads, dim", [(1, 4, 2, 128), (700, 8, 1, 64), (33_000, 8, 1, 128),
                                                          (17_000, 16, 2, 256), (70_001, 4, 1, 64)])
def test_no_requests(capi, cabi, tokens, heads, kv_heads, dim):
    """Every row is one of no request, however many there are; nothing is read of tables that have no entry."""
    query = torch.ones((tokens, heads, dim), dtype=torch.bfloat16, device=DEV)
    cache = torch.zeros((3, kv_heads, 2, 16, dim // 2), dtype=torch.uint8, device=DEV)
    scales = torch.zeros((3, kv_heads, 2, dim // 32, 16), dtype=torch.uint8, device=DEV)
    ints = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)
    out = torch.full_like(query, float("nan"))                         # what the allocator hands out again
    del out
    got, lse = capi.page_attention(query, cache, scales, ints(0, 4), ints(1), ints(0), return_lse=True)
    assert bool((got == 0).all()) and bool(lse.isneginf().all())

    # the C entry point, whose arrays may be null then
    lib = cabi.load()
    view = cabi.PagedCache(cache.data_ptr(), scales.data_ptr(), 3, cache.stride(0), scales.stride(0), kv_heads, dim, 16)
    size = lib.shmt_page_attention_scratch_bytes(tokens, heads, kv_heads, dim, 2, 0, 0)
    scratch = torch.full((size,), 255, dtype=torch.uint8, device=DEV)
    got.fill_(float("nan"))
    lse.fill_(0)
    rc = lib.shmt_page_attention(ctypes.byref(view), query.data_ptr(), heads * dim, dim, 2, tokens, heads, None, 0, 0, None,
                                 None, 4, 0, 0.1, 0, 0, 0, got.data_ptr(), lse.data_ptr(), scratch.data_ptr(), size,
                                 torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.shmt_last_error()
    torch.cuda.synchronize()
    assert bool((got == 0).all()) and bool(lse.isneginf().all())


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_more_items_than_one_round_of_the_list(capi, dim):
    """1,500 requests in the kernel for many rows: the list of items takes two rounds of 1,024, finding a workgroup's first
    item in it takes two of 512."""
    rng = np.random.default_rng(dim)
    q = rng.integers(1, 4, 1500)
    lens = q + rng.integers(0, 20, 1500)
    b = Batch(dim, lens, q, 2, 1, dim, 16, torch.bfloat16)
    _check(capi, b, max_query_len=2000)
    _check(capi, b, max_query_len=2000, window=5, sinks=1)


@pytest.mark.parametrize("dim, items", [(64, 518), (128, 518), (256, 780)])
def test_more_items_than_threads_without_a_list(capi, dim, items):
    """256 requests of two items and more: every workgroup counts them in two rounds of 512."""
    rng = np.random.default_rng(dim)
    q = np.full(256, 33)
    q[rng.permutation(256)[:6]] = 65
    assert (-(-q * 8 // (128 if dim == 256 else 256))).sum() == items
    lens = q + rng.integers(0, 9, 256)
    b = Batch(dim, lens, q, 8, 1, dim, 16, torch.bfloat16)
    _check(capi, b, window=20, sinks=2)
    got = [capi.page_attention(*b.args(), b.scale, max_query_len=hint, return_lse=True) for hint in (65, 1)]
    for x, y in zip(*got):                                             # the kernel for few rows counts otherwise; each within 2^-7
        assert bool(((x - y).abs() <= 2.0 ** -6 * (1 + y.abs())).all())
