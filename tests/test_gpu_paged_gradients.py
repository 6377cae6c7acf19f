"""The paged 4-bit cache gives no gradients, and says so."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_gradients_are_refused_not_lost(capi):
    cache = torch.zeros((2, 1, 2, 16, 32), dtype=torch.uint8, device=DEV)
    scales = torch.zeros((2, 1, 2, 2, 16), dtype=torch.uint8, device=DEV)
    slots = torch.arange(3, device=DEV)
    plain = torch.ones((3, 1, 64), dtype=torch.bfloat16, device=DEV)
    learned = plain.clone().requires_grad_()
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    attend = lambda q: capi.page_attention(q, cache, scales, ints(0, 1)[None], ints(0, 3), ints(3))
    for call in (lambda: capi.page_set(cache, scales, slots, learned, plain),
                 lambda: capi.page_set(cache, scales, slots, plain, learned),
                 lambda: capi.page_set(cache, scales, slots, plain, learned * 2),
                 lambda: attend(learned), lambda: attend(learned * 2)):
        with pytest.raises(RuntimeError, match="requires a gradient"):
            call()
    assert not bool(scales.any())
    with torch.no_grad():
        capi.page_set(cache, scales, slots, learned, plain)
        want = attend(learned)
    with torch.inference_mode():
        assert torch.equal(attend(plain), want)
    assert torch.equal(attend(learned.detach()), want) and bool((want == 1).all())
