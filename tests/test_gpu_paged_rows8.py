"""Rows rounded into a cache held in 8 bits, and read back: bit for bit what the definition says (oracle/paged_more.py). Rounding
to 8 bits is whole-number work, so there are no tolerances; reading rounds once more, to the type that is asked for."""
import numpy as np
import pytest
import torch

from oracle import paged_more

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _cache(pages, heads, page, dim, fill=None):
    cache = torch.zeros((pages, heads, 2, page, dim), dtype=torch.uint8)
    scales = torch.zeros((pages, heads, 2, dim // 32, page), dtype=torch.uint8)
    if fill is not None:
        cache.fill_(fill), scales.fill_(fill)
    return cache, scales


def _rows(gen, n, heads, dim, dtype, spread=0):
    x = torch.randn((n, heads, dim), generator=gen)
    if spread:
        x = x * torch.exp2(torch.randint(-spread, spread + 1, (n, heads, dim // 32), generator=gen).float()).repeat_interleave(32, -1)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page, heads, n", [(16, 1, 1), (16, 3, 37), (32, 8, 5), (64, 2, 200), (128, 1, 130), (256, 2, 700)])
def test_rows_as_defined(capi, dtype, dim, page, heads, n):
    gen = torch.Generator().manual_seed(n + dim)
    pages = -(-n // page) + 2
    keys, values = (_rows(gen, n, heads, dim, dtype, 12 if dtype == torch.float16 else 100) for _ in range(2))
    slots = torch.randperm(pages * page, generator=gen)[:n]
    slots[::7] = -1
    slots[3::11] = pages * page                                        # behind the cache: nowhere
    cache, scales = _cache(pages, heads, page, dim, 77)
    there = cache.to(DEV).view(torch.float8_e4m3fn), scales.to(DEV)
    capi.page_set(*there, slots.to(DEV), keys.to(DEV), values.to(DEV))
    paged_more.rows_set(cache.numpy(), scales.numpy(), slots.tolist(), keys.double().numpy(), values.double().numpy(), 8)
    assert torch.equal(there[0].view(torch.uint8).cpu(), cache) and torch.equal(there[1].cpu(), scales)
    for out in TYPES:
        for got, want in zip(capi.page_fetch(*there, slots.to(DEV), out),
                             paged_more.rows_fetch(cache.numpy(), scales.numpy(), slots.tolist(), 8)):
            want = torch.from_numpy(want).to(out)
            assert got.dtype == out and torch.equal(torch.nan_to_num(got.cpu(), nan=123), torch.nan_to_num(want, nan=123))


def test_edges_of_the_rounding(capi):
    """Ties, the largest and smallest numbers of 32 bits, zeros of both signs, what is not finite."""
    levels = torch.from_numpy(paged_more.LEVELS8)
    x = torch.zeros((40, 1, 64))
    mids = ((levels[:-1] + levels[1:]) / 2).float()                    # 126 ties, with 448 in front of each 31
    for i in range(5):
        part = mids[31 * i:31 * i + 31]
        x[i, 0, 0], x[i, 0, 1:1 + len(part)] = 448, part
        x[i, 0, 32], x[i, 0, 33:33 + len(part)] = -448, -part
        x[5 + i] = torch.nextafter(x[i], torch.zeros(()))
        x[10 + i] = torch.nextafter(x[i], torch.full((), 1e9))
    top = torch.finfo(torch.float32).max
    for i, v in enumerate([464, np.nextafter(np.float32(464), np.float32(0)), 463.99, 2.0 ** -126, 2.0 ** -149, -top, top, np.inf,
                           -np.inf, np.nan, -0.0, 2.0 ** -140, 448 * 2.0 ** -127, 1.8125 * 2.0 ** 127, 240 * 2.0 ** 120]):
        x[15 + i, 0, 5], x[15 + i, 0, 40] = float(v), float(v) / 3
    x[35, 0, :32] = -0.0
    cache, scales = _cache(3, 1, 16, 64)
    slots = torch.arange(40)
    there = cache.to(DEV).view(torch.float8_e4m3fn), scales.to(DEV)
    capi.page_set(*there, slots.to(DEV), x.to(DEV), (x * 2.0 ** -20).to(DEV))
    paged_more.rows_set(cache.numpy(), scales.numpy(), slots.tolist(), x.double().numpy(), (x * 2.0 ** -20).double().numpy(), 8)
    assert torch.equal(there[1].cpu(), scales)
    wrong = (there[0].view(torch.uint8).cpu() != cache).nonzero()
    assert len(wrong) == 0, wrong[:5]
    got = capi.page_fetch(*there, slots.to(DEV), torch.float32)[0].cpu()
    want = torch.from_numpy(paged_more.rows_fetch(cache.numpy(), scales.numpy(), slots.tolist(), 8)[0]).float()
    assert torch.equal(torch.nan_to_num(got, nan=7.0), torch.nan_to_num(want, nan=7.0))
    assert torch.equal(torch.signbit(got[35]), torch.signbit(want[35]))


def test_strides_types_of_slots_and_pages_apart(capi):
    gen = torch.Generator().manual_seed(5)
    joint = _rows(gen, 50, 9, 128, torch.bfloat16).to(DEV)
    keys, values = joint[:, 2:5], joint[:, 5:8]
    big = torch.zeros((5, 2, 3, 2, 16, 128), dtype=torch.uint8, device=DEV)
    scales = torch.zeros((5, 2, 3, 2, 4, 16), dtype=torch.uint8, device=DEV)
    plain = torch.zeros((5, 3, 2, 16, 128), dtype=torch.uint8, device=DEV), torch.zeros((5, 3, 2, 4, 16), dtype=torch.uint8, device=DEV)
    slots = torch.randperm(80, generator=gen)[:50].to(DEV)
    capi.page_set(big[:, 1].view(torch.float8_e4m3fn), scales[:, 1], slots.int(), keys, values)
    capi.page_set(plain[0].view(torch.float8_e4m3fn), plain[1], slots, keys.contiguous(), values.contiguous())
    assert torch.equal(big[:, 1], plain[0]) and torch.equal(scales[:, 1], plain[1]) and not bool(big[:, 0].any())
    odd = torch.zeros((50, 3, 131), dtype=torch.bfloat16, device=DEV)[..., 1:129]       # rows that begin anywhere are copied
    odd.copy_(keys)
    capi.page_set(big[:, 0].view(torch.float8_e4m3fn), scales[:, 0], slots, odd, values)
    assert torch.equal(big[:, 0], plain[0])


def test_refusals(capi):
    cache, scales = _cache(2, 1, 16, 64)
    cache, scales = cache.to(DEV).view(torch.float8_e4m3fn), scales.to(DEV)
    slots, rows = torch.arange(3, device=DEV), torch.ones((3, 1, 64), dtype=torch.bfloat16, device=DEV)
    for bad, text in ((lambda: capi.page_set(cache.view(torch.uint8).view(torch.float8_e5m2), scales, slots, rows, rows), "uint8"),
                      (lambda: capi.page_set(cache.view(torch.uint8), scales, slots, rows, rows), "scales must be"),
                      (lambda: capi.page_set(cache[..., :32], scales, slots, rows, rows), "64, 128 or 256"),
                      (lambda: capi.page_set(cache, scales, slots, rows[:2], rows), "keys and values"),
                      (lambda: capi.page_set(cache, scales, slots, rows.clone().requires_grad_(), rows), "requires a gradient"),
                      (lambda: capi.page_fetch(cache[:, :, :, ::2], scales[..., ::2], slots, torch.float32), "contiguous"),
                      (lambda: capi.page_fetch(cache, scales, slots, torch.int32), "dtype"),
                      (lambda: capi.page_fetch(cache, scales.cpu(), slots, torch.float32), "CUDA")):
        with pytest.raises(RuntimeError, match=text):
            bad()
    assert not bool(cache.view(torch.uint8).any()) and not bool(scales.any())
    assert [t.shape for t in capi.page_fetch(cache, scales, slots[:0], torch.float32)] == [(0, 1, 64)] * 2
