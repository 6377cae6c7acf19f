"""PagedCache queues its steps without waiting for the GPU."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_no_step_waits_for_the_gpu():
    import shmtensor_amd
    shmtensor_amd.install_aliases()
    from shmtensor_amd.shmtensor import PagedCache

    def run(cache, wait):
        """Six steps behind a kernel that takes its time; whether it was still running after each, and what came out."""
        gen = torch.Generator(device="cuda").manual_seed(1)
        rows = [torch.randn((12, h, 64), generator=gen, device="cuda").bfloat16() for h in (4, 2, 2)]
        torch.cuda.synchronize()
        done, behind, out = torch.cuda.Event(), [], []
        if wait:
            torch.cuda._sleep(2_000_000_000)                           # about a second
        done.record()
        for turn in range(6):
            new = np.array([9, 0, turn % 3, 1])
            step = cache.plan(new)
            q, k, v = (x[:step.tokens] for x in rows)
            cache.set(step, 0, k, v)
            out.append((cache.attend(step, 0, q, window=6, sinks=2), step.positions, step.slots, step.kv_lens))
            cache.trim(0, 6, 2)
            if turn == 3:
                cache.release(2)
            behind.append(not done.query())
        torch.cuda.synchronize()
        return behind, out

    make = lambda: PagedCache(pages=30, kv_heads=2, dim=64, requests=4, max_len=100)
    _, want = run(make(), wait=False)                                  # and all memory is at hand afterwards
    cache = make()
    behind, got = run(cache, wait=True)
    assert all(behind), behind
    assert cache.block_table[0, 1:3].tolist() == [-1, -1]                   # trim() gave pages back
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_more_steps_than_are_on_their_way():
    """Lengths of a step are not overwritten by those of a later one, however far the host is ahead."""
    import shmtensor_amd
    shmtensor_amd.install_aliases()
    from shmtensor_amd.shmtensor import PagedCache
    cache = PagedCache(pages=200, kv_heads=1, dim=64, requests=3, max_len=1000)
    cache.plan([0, 0, 0])
    torch.cuda.synchronize()
    torch.cuda._sleep(500_000_000)
    want, got = np.zeros(3, np.int64), []
    for turn in range(100):
        new = np.array([turn % 5, 1, (turn * 7) % 3])
        want = want + new
        got.append((cache.plan(new).kv_lens, want))
    for lens, total in got:
        assert lens.tolist() == total.tolist()
