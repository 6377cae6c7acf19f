"""More rows and heads in one call than one launch has threads for."""
import pytest
import torch

from oracle import paged

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_rows_beyond_one_launch(capi):
    heads, tokens = 65_535, 16_500                                     # 129 (or 258) x 64 tokens of 131,070 tiles: 2^32 and more
    cache = torch.zeros((1, heads, 2, 16, 32), dtype=torch.uint8, device=DEV)
    scales = torch.zeros((1, heads, 2, 2, 16), dtype=torch.uint8, device=DEV)
    gen = torch.Generator().manual_seed(0)
    keys, values = torch.randn((2, 1, heads, 64), generator=gen).bfloat16()
    slots = torch.full((tokens,), -1, dtype=torch.int64, device=DEV)
    for token, slot in ((0, 3), (8_150, 5), (8_200, 15), (16_499, 0)):
        slots[token] = slot
    wide = lambda x: x.to(DEV).expand(tokens, heads, 64)               # one row for all tokens
    capi.page_set(cache, scales, slots, wide(keys), wide(values))
    kept = (3, 5, 15, 0)
    for which, rows in enumerate((keys, values)):
        code, byte = (torch.from_numpy(x[0]) for x in paged.encode(rows.double().numpy()))
        packed = (code[:, 0::2] | code[:, 1::2] << 4).to(DEV)
        for slot in range(16):
            want = (packed, byte.to(DEV)) if slot in kept else (torch.zeros_like(packed), torch.zeros_like(byte).to(DEV))
            assert torch.equal(cache[0, :, which, slot], want[0]) and torch.equal(scales[0, :, which, :, slot], want[1]), slot
