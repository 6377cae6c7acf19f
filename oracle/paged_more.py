"""The paged cache's further operators in 64 bits and loops, as tests compare with (test infrastructure only): rows held in 8
bits, trees of drafted tokens, attention over either, the path that is kept. Written from the definitions in include/shmt.h;
oracle/paged.py has the 4-bit rows and the plan."""
import numpy as np

from oracle import paged

# the values of the codes 0 .. 126 (sign bit 0; 127 is not a number): 4 bits of exponent, 3 of mantissa
LEVELS8 = np.array([(m / 8 * 2.0 ** -6) if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])


def encode8(x):
    """(codes uint8 [..., dim], scale bytes [..., dim / 32]): the smallest power of two with max |x| < 464 2^e, e >= -127;
    values to the nearest level, ties to the even code."""
    x = np.asarray(x, dtype=np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    broken = ~np.isfinite(b).all(-1)
    b = np.where(broken[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    e = np.full(top.shape, -127)
    for step in (128, 64, 32, 16, 8, 4, 2, 1):                 # the largest e whose predecessor is too small
        e = np.where(top >= 464 * np.exp2(e + step - 1.0), e + step, e)
    y = np.abs(b) / np.exp2(e.astype(np.float64))[..., None]
    at = np.clip(np.searchsorted(LEVELS8, y, side="right") - 1, 0, 125)          # the level at or below, and the next one
    below, above = y - LEVELS8[at], LEVELS8[at + 1] - y
    code = np.where((above < below) | ((above == below) & (at % 2 == 1)), at + 1, at)
    code = np.where(broken[..., None], 0, code + 128 * np.signbit(b))
    return code.reshape(x.shape).astype(np.uint8), np.where(broken, 255, e + 127).astype(np.uint8)


def decode8(code, byte):
    v = np.append(LEVELS8, np.nan)[code & 127] * np.where(code & 128, -1.0, 1.0)
    s = np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))
    return (v.reshape(*byte.shape, 32) * s[..., None]).reshape(code.shape)


def rows_set(cache, scales, slots, keys, values, bits):
    """page_set on numpy arrays (uint8) of the cache's own layout, in place."""
    if bits == 4:
        return paged.rows_set(cache, scales, slots, keys, values)
    pages, page = cache.shape[0], cache.shape[3]
    for which, rows in enumerate((keys, values)):
        code, byte = encode8(rows)
        for i, s in enumerate(slots):
            if 0 <= s < pages * page:
                cache[s // page, :, which, s % page] = code[i]
                scales[s // page, :, which, :, s % page] = byte[i]


def rows_fetch(cache, scales, slots, bits):
    """float64 (keys, values) [slots, kv_heads, dim]; 0 where a slot is outside the cache."""
    if bits == 4:
        return paged.rows_fetch(cache, scales, slots)
    pages, heads, _, page, dim = cache.shape
    out = np.zeros((2, len(slots), heads, dim))
    for i, s in enumerate(slots):
        if 0 <= s < pages * page:
            out[:, i] = decode8(cache[s // page, :, :, s % page], scales[s // page, :, :, :, s % page]).transpose(1, 0, 2)
    return out[0], out[1]


def clean(parents):
    return [int(p) if 0 <= p < i else -1 for i, p in enumerate(parents)]


def tree(parents, starts, kv_lens):
    """(nodes [tokens, 4], positions [tokens]); -1 in rows of no request."""
    nodes, positions = np.full((len(parents), 4), -1, np.int64), np.full(len(parents), -1, np.int64)
    for b, length in enumerate(kv_lens):
        lo, hi = int(starts[b]), int(starts[b + 1])
        p = clean(parents[lo:hi])
        children = [[c for c in range(len(p)) if p[c] == i] for i in range(-1, len(p))]
        depth, order = {}, []
        todo = [(c, 0) for c in reversed(children[0])]
        while todo:
            i, d = todo.pop()
            order.append(i)
            depth[i] = d
            todo += [(c, d + 1) for c in reversed(children[i + 1])]
        for number, i in enumerate(order):
            size = 1
            while number + size < len(order) and depth[order[number + size]] > depth[i]:
                size += 1
            nodes[lo + i] = number, size, depth[i], min(depth[j] for j in range(i, len(p)))
            positions[lo + i] = length - len(p) + depth[i]
    return nodes, positions


def above(parents):
    """bool [n, n]: whether the second node is the first or an ancestor of it."""
    p, n = clean(parents), len(parents)
    out = np.zeros((n, n), bool)
    for i in range(n):
        j = i
        while j >= 0:
            out[i, j] = True
            j = p[j]
    return out


def keep(cache, scales, table, starts, kv_lens, parents, tokens, picked, given=None):
    """(counts, path, next); the rows of `cache` and `scales` ([layers, pages, ...]) are moved in place."""
    pages, page = cache.shape[1], cache.shape[4]
    counts, path, after = [], np.full(len(parents), -1, np.int64), []
    for b, length in enumerate(kv_lens):
        lo, hi = int(starts[b]), int(starts[b + 1])
        n = hi - lo
        if n == 0:
            counts.append(0)
            after.append(-1)
            continue
        mine = list(range(min(max(1 if given is None else int(given[b]), 1), n)))
        while True:
            at = mine[-1]
            fits = [c for c in range(at + 1, n) if parents[lo + c] == at and tokens[lo + c] == picked[lo + at]]
            if not fits:
                break
            mine.append(fits[0])
        path[lo:lo + len(mine)] = mine
        counts.append(len(mine))
        after.append(int(picked[lo + mine[-1]]))

        def slot(token):
            if token < 0 or token // page >= table.shape[1]:
                return None
            at = int(table[b, token // page])
            return (at, token % page) if 0 <= at < pages else None
        was = cache.copy(), scales.copy()
        for k, node in enumerate(mine):
            s, d = slot(int(length) - n + node), slot(int(length) - n + k)
            if k != node and s and d:
                cache[:, d[0], :, :, d[1]] = was[0][:, s[0], :, :, s[1]]
                scales[:, d[0], :, :, :, d[1]] = was[1][:, s[0], :, :, :, s[1]]
    return np.array(counts), path, np.array(after)


def attention(query, cache, scales, table, starts, kv_lens, scale, bits=4, seen="causal", parents=None, window=0, sinks=0):
    """(out, lse, spread, top), as oracle.paged.attention has them. seen: "causal", "tree" (with parents) or "all"."""
    tokens, heads, dim = query.shape
    pages, kv_heads, _, page, _ = cache.shape
    out, spread = np.zeros(query.shape), np.zeros(query.shape)
    lse, top = np.full((tokens, heads), -np.inf), np.zeros((tokens, heads))
    for b, length in enumerate(kv_lens.tolist()):
        lo, hi = int(starts[b]), int(starts[b + 1])
        where = table[b].repeat(page).astype(np.int64)
        j = np.nonzero((where >= 0) & (where < pages) & (np.arange(len(where)) < length))[0]
        k, v = rows_fetch(cache, scales, where[j] * page + j % page, bits)
        first = length - (hi - lo)
        mine = above(parents[lo:hi]) if seen == "tree" else None
        depth = mine.sum(1) - 1 if seen == "tree" else None
        for t in range(lo, hi):
            if seen == "all":
                sees, place, p = np.ones(len(j), bool), j, length - 1
            elif seen == "causal":
                p = first + t - lo
                sees, place = j <= p, j
            else:
                p = first + depth[t - lo]
                node = np.clip(j - first, 0, hi - lo - 1)
                sees = (j < first) | mine[t - lo, node]
                place = np.where(j < first, j, first + depth[node])
            if window:
                sees = sees & ((place > p - window) | (place < sinks))
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
