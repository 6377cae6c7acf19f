"""The definitions that the GPU tests of trees, 8-bit rows and attention over them compare with, held to simpler statements."""
import numpy as np
import torch

from oracle import paged, paged_more


def test_8_bit_levels_are_those_of_the_type():
    want = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(paged_more.LEVELS8, want)


def test_8_bit_rows_round_to_the_nearest_level():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((200, 64)) * np.exp2(rng.integers(-120, 110, (200, 1)))
    x[0], x[1, :32], x[2, 5] = 0, 464, np.inf
    x[3, :32], x[3, 32:] = 463.9, np.nextafter(464, 0)
    code, byte = paged_more.encode8(x)
    y = paged_more.decode8(code, byte)
    assert (byte[0] == 0).all() and (y[0] == 0).all() and byte[1, 0] == 128 and byte[2, 0] == 255 and np.isnan(y[2, :32]).all()
    assert (byte[3] == 127).all() and (code[3] == 126).all()
    fine = np.isfinite(y)
    top = np.abs(np.where(np.isfinite(x), x, 0)).reshape(200, 2, 32).max(-1).repeat(32, 1).reshape(x.shape)
    # half a step: 2^-4 of the value, or 2^-10 of the scale, which is below 2^-8 of the largest over 1.8
    assert (np.abs(x - y)[fine] <= (np.abs(x) * 2.0 ** -4 + top * 2.0 ** -18 + 2.0 ** -137)[fine]).all()
    far = torch.tensor(x / np.exp2(byte.astype(float) - 127).repeat(32, 1).clip(1e-300)).float()
    with np.errstate(invalid="ignore"):
        ours = torch.from_numpy(code[4:]).view(torch.float8_e4m3fn).float()
    assert torch.equal(far[4:].clamp(-448, 448).to(torch.float8_e4m3fn).float(), ours)


def test_ties_go_to_the_even_code():
    x = np.zeros((1, 32))
    mids = (paged_more.LEVELS8[:-1] + paged_more.LEVELS8[1:]) / 2
    x = np.concatenate([mids, np.full(2, 448.0)]).reshape(4, 32)
    x[:, 0] = 448.0                                            # every block has the power of two 1
    code, byte = paged_more.encode8(x)
    assert (byte == 127).all() and (code.reshape(-1)[1:126] % 2 == 0)[np.arange(1, 126) % 32 != 0].all()


def test_numbers_and_sizes_say_who_is_above():
    rng = np.random.default_rng(1)
    for n in (1, 2, 7, 40):
        parents = [int(rng.integers(-1, i)) if i else -1 for i in range(n)]
        nodes, positions = paged_more.tree(parents, [0, n], [n + 3])
        gap = nodes[:, 0][:, None] - nodes[:, 0][None, :]
        assert np.array_equal((gap >= 0) & (gap < nodes[:, 1][None, :]), paged_more.above(parents))
        assert sorted(nodes[:, 0]) == list(range(n)) and np.array_equal(positions, nodes[:, 2] + 3)
        assert np.array_equal(nodes[:, 2], paged_more.above(parents).sum(1) - 1)


def test_a_chain_is_causal():
    rng = np.random.default_rng(2)
    cache, scales = rng.integers(0, 256, (6, 1, 2, 16, 32), np.uint8), rng.integers(120, 128, (6, 1, 2, 2, 16)).astype(np.uint8)
    table, starts, lens = np.array([[3, 1, 0]]), np.array([0, 5]), np.array([40])
    q = rng.standard_normal((5, 2, 64))
    for window, sinks in ((0, 0), (7, 2)):
        kw = dict(window=window, sinks=sinks)
        want = paged.attention(q, cache, scales, table, starts, lens, 0.1, **kw)
        chain = paged_more.attention(q, cache, scales, table, starts, lens, 0.1, seen="tree", parents=[-1, 0, 1, 2, 3], **kw)
        causal = paged_more.attention(q, cache, scales, table, starts, lens, 0.1, **kw)
        for a, b, c in zip(want, chain, causal):
            assert np.array_equal(a, b) and np.array_equal(a, c)
    every = paged_more.attention(q[4:], cache, scales, table, np.array([0, 1]), lens, 0.1, seen="all")
    assert np.array_equal(every[0], paged.attention(q, cache, scales, table, starts, lens, 0.1)[0][4:])


def test_kept_rows_are_read_before_their_places_are_written():
    cache = np.arange(16, dtype=np.uint8).reshape(1, 1, 1, 1, 16, 1).repeat(2, 3).copy()
    scales = cache.transpose(0, 1, 2, 3, 5, 4).copy()
    counts, path, after = paged_more.keep(cache, scales, np.array([[0]]), [0, 6], [8], [-1, 0, 0, 2, 3, 4],
                                          [9, 5, 1, 2, 3, 4], [1, 7, 2, 3, 4, 8])
    assert counts.tolist() == [5] and path.tolist() == [0, 2, 3, 4, 5, -1] and after.tolist() == [8]
    want = [0, 1, 2, 4, 5, 6, 7, 7] + list(range(8, 16))
    assert cache[0, 0, 0, 0, :, 0].tolist() == want and scales[0, 0, 0, 1, 0].tolist() == want
