"""The paged key/value cache held in 4 bits, in 64 bits and loops: the definition that the GPU operators are tested
against (test infrastructure only). Rows are numpy arrays; 16-bit floats come as float64 of the same values."""
import numpy as np

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def encode(x):
    """(codes [..., dim], scale bytes [..., dim / 32]) of rows. A block's power of two is the smallest with
    max |x| < 7 * 2^e, e >= -127; values go to the nearest level, ties to the even code."""
    x = np.asarray(x, dtype=np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    broken = ~np.isfinite(b).all(-1)
    top = np.where(broken, 1.0, np.abs(np.where(np.isfinite(b), b, 0)).max(-1))
    e = np.full(top.shape, -127)
    for step in (128, 64, 32, 16, 8, 4, 2, 1):                 # the largest e whose predecessor is too small
        e = np.where(top >= 7 * np.exp2(e + step - 1.0), e + step, e)
    y = np.abs(np.where(broken[..., None], 0, b)) / np.exp2(e.astype(np.float64))[..., None]
    far = np.abs(y[..., None] - LEVELS)
    near = far == far.min(-1, keepdims=True)
    first = near.argmax(-1)                                    # at a tie two neighbours are near: the even one
    code = np.where((near.sum(-1) == 2) & (first % 2 == 1), first + 1, first)
    code = np.where(broken[..., None], 0, code + 8 * np.signbit(b))
    return code.reshape(x.shape).astype(np.uint8), np.where(broken, 255, e + 127).astype(np.uint8)


def decode(code, byte):
    """float64 rows from codes and scale bytes; NaN where the byte is 255."""
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))
    return (v.reshape(*byte.shape, 32) * s[..., None]).reshape(code.shape)


def rows_set(cache, scales, slots, keys, values):
    """page_set on numpy arrays of the cache's own layout, in place."""
    pages, _, _, page, _ = cache.shape
    for which, rows in enumerate((keys, values)):
        code, byte = encode(rows)
        packed = code[..., 0::2] | code[..., 1::2] << 4
        for i, s in enumerate(slots):
            if 0 <= s < pages * page:
                cache[s // page, :, which, s % page] = packed[i]
                scales[s // page, :, which, :, s % page] = byte[i]


def rows_fetch(cache, scales, slots):
    """float64 (keys, values) [slots, kv_heads, dim]; 0 where a slot is outside the cache."""
    pages, heads, _, page, half = cache.shape
    out = np.zeros((2, len(slots), heads, 2 * half))
    for i, s in enumerate(slots):
        if 0 <= s < pages * page:
            packed = cache[s // page, :, :, s % page]
            code = np.stack([packed & 15, packed >> 4], -1).reshape(heads, 2, 2 * half)
            out[:, i] = decode(code, scales[s // page, :, :, :, s % page]).transpose(1, 0, 2)
    return out[0], out[1]


def plan(cached, new, table, free, page, max_tokens):
    """(query_starts, kv_lens, positions, slots, counts); `table` is extended in place."""
    cached, new = np.maximum(cached, 0), np.maximum(new, 0)
    starts, positions, slots, taken = [0], [], [], 0
    width = table.shape[1]
    for b, (c, n) in enumerate(zip(cached.tolist(), new.tolist())):
        for p in range(-(-c // page), -(-(c + n) // page)):
            if p < width:
                table[b, p] = free[taken] if taken < len(free) else -1
            taken += 1
        for pos in range(c, c + n):
            at = table[b, pos // page] if pos // page < width else -1
            positions.append(pos)
            slots.append(at * page + pos % page if at >= 0 else -1)
        starts.append(starts[-1] + n)
    counts = [starts[-1], taken]
    room = [-1] * max(0, max_tokens - len(slots))
    return (np.array(starts, np.int32), (cached + new).astype(np.int32), np.array((positions + room)[:max_tokens], np.int32),
            np.array((slots + room)[:max_tokens], np.int64), np.array(counts, np.int64))


def attention(query, cache, scales, table, starts, kv_lens, scale, window=0, sinks=0):
    """(out, lse, spread, top): attention in float64; per row and head also sum_j w_j |V_j| and the largest
    scale * sum_d |q_d K_jd|, from which error bounds follow."""
    tokens, heads, dim = query.shape
    pages, kv_heads, _, page, _ = cache.shape
    out, spread = np.zeros(query.shape), np.zeros(query.shape)
    lse, top = np.full((tokens, heads), -np.inf), np.zeros((tokens, heads))
    for b, length in enumerate(kv_lens.tolist()):
        lo, hi = int(starts[b]), int(starts[b + 1])
        where = table[b].repeat(page).astype(np.int64)
        j = np.nonzero((where >= 0) & (where < pages) & (np.arange(len(where)) < length))[0]
        k, v = rows_fetch(cache, scales, where[j] * page + j % page)
        for t in range(lo, hi):
            p = length - (hi - lo) + t - lo
            sees = j <= p
            if window:
                sees &= (j > p - window) | (j < sinks)
            if not sees.any():
                continue
            for h in range(heads):
                kk, vv = k[sees, h * kv_heads // heads], v[sees, h * kv_heads // heads]
                s = kk @ query[t, h] * scale
                top[t, h] = (np.abs(kk) @ np.abs(query[t, h])).max() * abs(scale)
                m = s.max()
                w = np.exp(s - m)
                lse[t, h] = m + np.log(w.sum())
                w /= w.sum()
                out[t, h], spread[t, h] = w @ vv, w @ np.abs(vv)
    return out, lse, spread, top
