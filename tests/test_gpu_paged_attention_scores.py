"""Attention over the paged 4-bit cache where scores are large: far above those that a row sees first, or so far from 0 that a
float's last place is more than an exponent of 2 can move by. Against the definition in 64 bits (oracle/paged.py).

Queries have one dimension that is not 0 and keys hold few bits, so scores are exact before they are scaled and tokens with
the greatest one are tied exactly. Scaling rounds a score by 2^-21 of itself at most, which moves the weights of other tokens by
that part; from 2^12 on there are none that are not 0 (the next level of a key is a quarter less at least). Bounds are those of
test_gpu_paged_attention.py otherwise."""
import numpy as np
import pytest
import torch

from test_gpu_paged_attention import Batch, _check, _close

pytestmark = pytest.mark.gpu

ROWS = [([90, 300, 17, 1000], [1, 1, 1, 1], 0), ([150, 70, 200], [5, 3, 7], 7), ([300, 40, 130], [290, 1, 70], 4000)]


def _one_dimension(batch, at):
    """Queries that are not 0 in dimension `at` only."""
    q = torch.zeros_like(batch.query)
    q[..., at] = batch.query[..., at].abs().clamp(0.5, 2.0) * torch.where(batch.query[..., at] < 0, -1.0, 1.0).to(q.dtype)
    batch.query = q


def _exact(capi, batch, hint, **kw):
    out, lse, spread, top = batch.want(**kw)
    assert np.isfinite(out).all() and np.isfinite(lse).all()
    got, got_lse = capi.page_attention(*batch.args(), batch.scale, max_query_len=hint, return_lse=True, **kw)
    dim = batch.query.shape[2]
    allowed = 8.0 / (dim + 8) * np.minimum(top, 2.0 ** 12)             # as _close counts: (dim + 8) 2^-24 of it
    _close(got, None, (out, lse, spread, allowed), batch.query.dtype, dim)
    l = got_lse.double().cpu().numpy()
    assert (np.abs(l - lse) <= 2.0 ** -15 + 2.0 ** -20 * np.abs(lse)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", range(len(ROWS)))
@pytest.mark.parametrize("power", [18, 24, 29, 30, 31, 33, 40, 63, 90, 120])
def test_scores_of_any_size_end_and_are_right(capi, power, rows, dim, dtype):
    lens, q, hint = ROWS[rows]
    b = Batch(power + dim + rows, lens, q, 6, 2, dim, 16, dtype)
    _one_dimension(b, 40)
    live = b.scales[:, :, 0] != 255
    b.scales[:, :, 0] = torch.where(live, torch.tensor(127 + power, dtype=torch.uint8), b.scales[:, :, 0])
    b.scale = -0.3 if power % 2 else 0.3
    _exact(capi, b, hint)
    _exact(capi, b, hint, window=60, sinks=9)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", range(len(ROWS)))
@pytest.mark.parametrize("tokens_a_step, first", [(1, -40), (8, -10), (40, 3)])
def test_scores_that_grow_with_every_token(capi, tokens_a_step, first, rows, dim, dtype):
    """Every tile's scores are far above those of the tile before it."""
    lens, q, hint = ROWS[rows]
    b = Batch(tokens_a_step + dim + rows, lens, q, 4, 1, dim, 16, dtype)
    _one_dimension(b, 3)
    b.query.abs_()
    b.cache[:, :, 0, :, 1] = b.cache[:, :, 0, :, 1] & 15 | 0x20        # dimension 3: 1
    for r, n in enumerate(lens):
        j = torch.arange(n)
        at, off = b.table[r, j // 16].long(), j % 16
        b.scales[at, 0, 0, 0, off] = (127 + first + j // tokens_a_step).clamp(max=240).byte()
    b.scale = 0.7
    _exact(capi, b, hint)
    _exact(capi, b, hint, window=100)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", range(len(ROWS)))
@pytest.mark.parametrize("power", [10, 20, 26, 30, 34, 50, 100])
def test_ordinary_rows_with_enormous_scores_stay_finite(capi, power, rows, dim, dtype):
    lens, q, hint = ROWS[rows]
    b = Batch(power, lens, q, 4, 2, dim, 16, dtype)
    live = b.scales[:, :, 0] != 255
    b.scales[:, :, 0][live] += power
    got, _ = _check(capi, b, max_query_len=hint)
    assert bool(got.isfinite().all())
    assert float(got.abs().max()) <= 6.0 * 1.01                        # values are 6 at most: weights sum up to 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", range(len(ROWS)))
@pytest.mark.parametrize("levels", [(2,), (4,), (2, 4, 6), (6, 2)])
@pytest.mark.parametrize("lead", [20, 25, 45, 64, 130, 1100, 3000])
def test_a_few_tokens_far_above_all_others(capi, lead, levels, rows, dim, dtype):
    """One token, or one after another, lead by 2^20 to 2^18,000: what one raise of the reference settles, what a second one
    would have to, sums beyond the floats, references far from 0."""
    lens, q, hint = ROWS[rows]
    b = Batch(lead + dim + rows, lens, q, 4, 2, dim, 16, dtype)
    b.query[:] = 0
    b.query[..., 2] = 1
    b.cache[:, :, 0, :, 1] = b.cache[:, :, 0, :, 1] & 0xF0             # dimension 2 of every key: 0
    b.scales[:, :, 0, 0] = torch.where(b.scales[:, :, 0, 0] != 255, torch.tensor(127, dtype=torch.uint8), b.scales[:, :, 0, 0])
    for r, n in enumerate(lens):
        for i, level in enumerate(levels):
            j = int(n * (0.5 + 0.4 * i / len(levels)))
            b.cache[int(b.table[r, j // 16]), :, 0, j % 16, 1] |= {2: 4, 4: 6, 6: 7}[level]
    b.scale = lead / 2 * np.log(2)
    _exact(capi, b, hint)
    _exact(capi, b, hint, window=200, sinks=3)


@pytest.mark.parametrize("requests, q, group, kv_heads", [(32, 1, 4, 8), (16, 7, 3, 8), (8, 180, 3, 1)])
def test_a_constant_in_all_scores_costs_nothing(capi, requests, q, group, kv_heads):
    """A score's distance from 0 is nothing that a softmax depends on. Items have lanes that hold no row (12 of 16, 11 of 32,
    the most of the last 256): what those make of scores must not send the item's rows through their tokens again, which takes
    half as long again at least. A quarter is allowed, of the least of many times, three times over."""
    b = Batch(1, [4000] * requests, [q] * requests, group * kv_heads, kv_heads, 128, 16, torch.bfloat16)
    b.cache[:, :, 0, :, 0] = b.cache[:, :, 0, :, 0] & 0xF0 | 2         # dimension 0 of every key: 1
    live = b.scales[:, :, 0, 0] != 255
    b.scales[:, :, 0, 0] = torch.where(live, torch.tensor(127, dtype=torch.uint8), b.scales[:, :, 0, 0])
    args = b.args()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)

    def least(constant):
        args[0][..., 0] = constant / b.scale
        times = []
        for _ in range(30):
            begin.record()
            for _ in range(10):
                capi.page_attention(*args, b.scale, max_query_len=q)
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times)

    least(0)
    pairs = [(least(0), least(40)) for _ in range(3)]
    assert any(far < 1.25 * near for near, far in pairs), pairs
