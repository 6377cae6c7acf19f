"""Attention over the paged cache of trees, of an encoder's states and over 8 bits: weights meet the values in 16 bits in both
kernels, so the hint `max_query_len` changes a result by less than its rounding. Bounds of test_gpu_paged_attention_weights.py:
2^-16 of each weight, and one rounding of the result."""
import numpy as np
import pytest
import torch

from test_gpu_paged_attention_seen import RULES, Batch
from test_gpu_paged_attention_weights import _close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits, seen", RULES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_the_hint_does_not_cost_bits(capi, bits, seen, dtype, dim):
    b = Batch(dim, [700, 90, 5, 333, 260], [70, 90, 5, 1, 129], 6, 2, dim, 16, dtype, bits, seen)
    rule = b.rule(capi)
    for kw in [{}] + ([dict(window=60, sinks=3)] if seen != "all" else []):
        want = b.want(**kw)
        for hint in (1, 5, 0, 100000):
            _close(capi.page_attention(*b.args(), b.scale, max_query_len=hint, **rule, **kw), want, dtype, dim)


@pytest.mark.parametrize("bits, seen", RULES)
def test_many_rows_over_long_requests(capi, bits, seen):
    """Items that several workgroups share."""
    b = Batch(3, [5000, 2100], [150, 64], 4, 1, 128, 32, torch.bfloat16, bits, seen, kinds=("late", "tree"))
    got = capi.page_attention(*b.args(), b.scale, max_query_len=150, **b.rule(capi))
    _close(got, b.want(), torch.bfloat16, 128)
    assert np.isfinite(got.float().cpu().numpy()).all()
