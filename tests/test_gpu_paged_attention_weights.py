"""Attention over the paged 4-bit cache for few rows a request: weights meet the values in 16 bits, whatever the queries' type.

Bounds of test_gpu_paged_attention.py, but for the weights: each is within 2^-16 of itself, so 2^-16 sum_j w_j |V_j| in all. The
round-off of a result is 2^-8 of it in bfloat16 and 2^-11 in float16."""
import numpy as np
import pytest
import torch

from test_gpu_paged_attention import TINY, Batch

pytestmark = pytest.mark.gpu
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _close(got, want, dtype, dim):
    out, _, spread, top = want
    score = ((dim + 8) * 2.0 ** -24 * top)[..., None]
    bound = ROUND[dtype] * np.abs(out) * (1 + 2.0 ** -7) + 2 * TINY[dtype] + (2.0 ** -16 + 4 * score + 2.0 ** -15) * spread
    far = np.abs(got.double().cpu().numpy() - out) - bound
    assert far.max() <= 0, "%.3g over its bound, %d of %d" % (far.max(), (far > 0).sum(), far.size)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads, kv_heads, q", [(4, 1, 1), (8, 2, 3), (6, 2, 9), (40, 1, 1)])
def test_results_are_off_by_little_more_than_their_rounding(capi, heads, kv_heads, q, dim, dtype):
    lens = [9, 20, 300, 77, 1200, 33]
    b = Batch(heads + dim, lens, [q] * 6, heads, kv_heads, dim, 16, dtype)
    for kw in ({}, dict(window=40, sinks=2)):
        _close(capi.page_attention(*b.args(), b.scale, max_query_len=q, **kw), b.want(**kw), dtype, dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("requests, length, q, group, kv_heads", [(8, 4000, 1, 4, 8), (4, 4000, 7, 3, 8)])
def test_a_token_that_has_all_the_weight_gives_its_value(capi, requests, length, q, group, kv_heads, dim, dtype):
    """A late token leads by 2^24.5 to 2^36.8 over all others, which were the reference before it came: its weight is no power
    of two, and its value comes out all the same."""
    b = Batch(dim + q, [length] * requests, [q] * requests, group * kv_heads, kv_heads, dim, 16, dtype)
    size = b.query[..., 7].float().abs()
    b.query[:] = 0
    b.query[..., 7] = (1 + size.frac() / 2).to(dtype)
    b.cache[:, :, 0, :, 3] = b.cache[:, :, 0, :, 3] & 0x0F | 0x10      # dimension 7 of every key: 0.5
    live = b.scales[:, :, 0, 0] != 255
    b.scales[:, :, 0, 0] = torch.where(live, torch.tensor(127, dtype=torch.uint8), b.scales[:, :, 0, 0])
    rng = np.random.default_rng(dim)
    for r in range(requests):
        for h in range(kv_heads):
            j = int(rng.integers(length // 2, length - q))
            page = b.cache[int(b.table[r, j // 16]), h, 0, j % 16]
            page[3] = page[3] & 0x0F | 0x70                            # 6
    b.scale = 24.5 / (5.5 * np.log2(np.e))
    _close(capi.page_attention(*b.args(), b.scale, max_query_len=q), b.want(), dtype, dim)
