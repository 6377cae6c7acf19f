"""Performance cases of the paged key/value cache's further operators: trees of drafted tokens, an encoder's states, 8 bits.

A program that drafts several continuations at once gives each request a tree of new tokens: node i's parent is a node
before it, or -1. Once a step the trees are numbered (`tree`), in every layer the nodes' queries attend to what the request
holds and to their own ancestors (`attend`, seen "tree"), and in the end the path that the model agrees with is kept, its
rows moved to where they would lie without the rest of the tree (`keep`). A decoder beside an encoder attends to all of a
request's states (`attend`, seen "all"). And a cache may be held in 8 bits instead of 4 (`rows`, `attend`).

In 8 bits a row of `dim` values is held as floats of 8 bits (sign, 4 bits of exponent, 3 of mantissa, up to 448) with one
power of two for every 32 values; in 4 bits (sign, 2, 1: 0, 0.5, 1, 1.5, 2, 3, 4, 6), the even dimension in the low bits:

    cache   float8_e4m3fn [pages, kv_heads, 2, page, dim], uint8 [pages, kv_heads, 2, page, dim / 2]    keys 0, values 1
    scales  uint8 [pages, kv_heads, 2, dim / 32, page]   2^(byte - 127); 255 stands for "not a number"

A node of a numbered tree is four words: its number when every node comes before its children and those in their order, the
size of its subtree, its depth, the least depth from it to the request's last node. An ancestor of node i is a node j with
0 <= number[i] - number[j] < size[j].
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "i32": torch.int32, "i64": torch.int64}
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
FLOAT8 = torch.float8_e4m3fn


def listed():
    return [
        # The trees of a handful of requests: latency only.
        dict(name="tree_few", kind="tree", requests=6, new_lo=1, new_hi=16, prompts=0.0, longest=0, dtype="i32"),
        # A full batch, trees of up to 64 nodes, some requests that bring a prompt (a tree that is a chain) instead.
        dict(name="tree_batch", kind="tree", requests=501, new_lo=1, new_hi=64, prompts=0.04, longest=400, dtype="i32"),
        # One user, two layers, 4 bits: latency only.
        dict(name="keep_few", kind="keep", requests=3, new_lo=7, new_hi=16, cached_lo=20, cached_hi=90, layers=2,
             kv_heads=8, dim=128, bits=4, page=16, dtype="i64"),
        # A full batch, all layers at once, 8 bits.
        dict(name="keep_batch", kind="keep", requests=120, new_lo=24, new_hi=64, cached_lo=1, cached_hi=90, layers=16,
             kv_heads=8, dim=128, bits=8, page=32, dtype="i64"),
        # The rows of one decode step, 8 bits.
        dict(name="rows8_decode", kind="rows", tokens=61, kv_heads=8, dim=128, bits=8, page=16, skip=0.05, dtype="bf16"),
        # Long prompts in 8 bits: the rows of 60 K tokens, slices of a joint projection.
        dict(name="rows8_prompts", kind="rows", tokens=60_001, kv_heads=8, dim=128, bits=8, page=64, skip=0.0,
             dtype="bf16"),
        # One user, nine drafted tokens, a short context: latency only.
        dict(name="tree_attend_one", kind="attend", seen="tree", requests=1, cached_lo=901, cached_hi=901, new_lo=9,
             new_hi=9, kv_heads=8, group=4, dim=128, bits=4, page=16, window=0, sinks=0, dtype="bf16"),
        # A full batch of ragged requests, 24 to 64 drafted tokens each.
        dict(name="tree_attend_batch", kind="attend", seen="tree", requests=40, cached_lo=1000, cached_hi=12_000,
             new_lo=24, new_hi=64, kv_heads=8, group=4, dim=128, bits=4, page=16, window=0, sinks=0, dtype="bf16"),
        # One long document in 8 bits, a tree of 13 tokens: the work has to be split over the cache.
        dict(name="tree_attend_long", kind="attend", seen="tree", requests=1, cached_lo=100_001, cached_hi=100_001,
             new_lo=13, new_hi=13, kv_heads=8, group=5, dim=128, bits=8, page=32, window=0, sinks=0, dtype="f16"),
        # Five hypotheses of each of 80 requests, a token each, over the encoder's states; every head its own keys.
        dict(name="cross_beams", kind="attend", seen="all", requests=80, cached_lo=300, cached_hi=1500, new_lo=5,
             new_hi=5, kv_heads=16, group=1, dim=64, bits=4, page=16, window=0, sinks=0, dtype="f16"),
        # Whole answers that are scored at once, over the encoder's states in 8 bits.
        dict(name="cross_answers8", kind="attend", seen="all", requests=6, cached_lo=700, cached_hi=5000, new_lo=100,
             new_hi=1200, kv_heads=8, group=2, dim=128, bits=8, page=64, window=0, sinks=0, dtype="bf16"),
        # A decode step of a full batch of ragged requests, 8 bits.
        dict(name="attend8_batch", kind="attend", seen="causal", requests=64, cached_lo=1000, cached_hi=16_000, new_lo=1,
             new_hi=1, kv_heads=8, group=4, dim=128, bits=8, page=16, window=0, sinks=0, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    kind = rng.choice(["tree", "keep", "rows", "attend", "attend", "attend", "attend"])
    page, bits = rng.choice([16, 32, 64, 128]), rng.choice([4, 8])
    heads, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 128, 256])
    if kind == "tree":
        prompts = rng.choice([0.0, 0.0, 0.1])
        longest = _log_int(rng, 65, 600) if prompts else 0
        n = _log_int(rng, 1, 60 if prompts else 500)
        new_hi = _log_int(rng, 1, 64) if rng.random() < 0.7 else _log_int(rng, 1, max(1, 12_000 // n) if n > 24 else 500)
        return dict(kind=kind, requests=n, new_lo=rng.choice([0, 1, new_hi]), new_hi=new_hi, prompts=prompts,
                    longest=longest, dtype=rng.choice(["i32", "i64"]))
    if kind == "keep":
        n, layers, new_hi = _log_int(rng, 1, 120), _log_int(rng, 1, 16), _log_int(rng, 1, 64)
        return dict(kind=kind, requests=n, new_lo=rng.choice([1, max(1, new_hi // 2)]), new_hi=new_hi, cached_lo=0,
                    cached_hi=rng.choice([0, 17, 90]), layers=layers, kv_heads=heads, dim=min(dim, 128), bits=bits,
                    page=min(page, 64), dtype=rng.choice(["i32", "i64"]))
    if kind == "rows":
        return dict(kind=kind, tokens=_log_int(rng, 1, 30_000), kv_heads=heads, dim=dim, bits=8, page=page,
                    skip=rng.choice([0.0, 0.02, 0.3]), dtype=rng.choice(["bf16", "f16", "f32"]))
    seen = rng.choice(["tree", "tree", "all", "causal"])
    bits = 8 if seen == "causal" else bits                  # (in 4 bits that is another file's)
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    few = seen == "tree" or rng.random() < 0.6
    n = _log_int(rng, 1, 96 if few else 6)
    new_hi = _log_int(rng, 1, 64) if seen == "tree" else rng.randint(1, 9) if few else _log_int(rng, 10, 2000)
    cached_hi = _log_int(rng, 1, max(1, min(100_000, 300_000_000 // (n * heads * dim))))
    rows = n * heads * group * new_hi
    cached_hi = max(1, min(cached_hi, 500_000_000 // rows))
    new_hi = min(new_hi, max(1, 500_000_000 // (n * heads * group * (cached_hi + new_hi))))
    window = 0 if seen == "all" else rng.choice([0, 0, _log_int(rng, 1, 8000)])
    return dict(kind=kind, seen=seen, requests=n, cached_lo=rng.choice([0, min(cached_hi, 20), max(1, cached_hi // 8)]),
                cached_hi=cached_hi, new_lo=rng.choice([1, max(1, new_hi // 4)]), new_hi=new_hi, kv_heads=heads,
                group=group, dim=dim, bits=bits, page=page, window=window,
                sinks=rng.choice([0, 1, 4, 37]) if window else 0, dtype=rng.choice(["bf16", "f16"]))


def _lengths(case):
    """(cached, new) of each request: spread over their ranges (by their logarithm), the same for every seed."""
    def spread(lo, hi, step):
        at = np.mod((np.arange(case["requests"]) + 0.5) * step, 1.0)
        return np.rint((lo + 1) * ((hi + 1) / (lo + 1)) ** at - 1).astype(np.int64)
    new = spread(case["new_lo"], case["new_hi"], 0.7548776662)
    if case["kind"] == "tree":
        new[:int(case["prompts"] * case["requests"])] = case["longest"]
        return spread(0, 4000, 0.6180339887), new
    return spread(case["cached_lo"], case["cached_hi"], 0.6180339887), new


def _pages(tokens, page):
    return -(-tokens // page)


def _seen(case, cached, new):
    """(tokens that some row of the request sees, pairs of a row and a token that it sees), per request; of a tree, whose
    pairs are its own, those of half a chain."""
    total, w, s = cached + new, case["window"], case["sinks"]
    if case["seen"] == "all":
        return cached, new * cached
    own_pairs = new * (new + 1) // (2 if case["seen"] == "causal" else 4)
    if not w:
        return total, new * cached + own_pairs
    first = np.maximum(cached - w + 1, 0)                     # the first row's window begins here
    tokens = np.minimum(total, s) + total - np.maximum(first, np.minimum(total, s))
    row = np.minimum(cached, w) + np.minimum(first, s)        # about what a row sees
    return np.where(new > 0, tokens, 0), new * row


def _row_bytes(case):
    return case["dim"] * case["bits"] // 8 + case["dim"] // 32


def work(case):
    """The bytes and the operations of one pass that nothing can do without."""
    if case["kind"] == "rows":
        values = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * (values * size + values + values // 32 + 8 * case["tokens"]), "flops": 2 * values}
    cached, new = _lengths(case)
    if case["kind"] == "tree":
        size = 4 if case["dtype"] == "i32" else 8
        return {"bytes": int(24 * new.sum() + (2 * case["requests"] + 1) * size), "flops": int(4 * new.sum())}
    if case["kind"] == "keep":                                # about two moved rows a request
        size = 4 if case["dtype"] == "i32" else 8
        rows = 2 * case["requests"] * case["layers"] * case["kv_heads"] * 2
        return {"bytes": int(2 * rows * _row_bytes(case) + new.sum() * (2 * size + 8) + case["requests"] * (size + 12)),
                "flops": int(2 * new.sum())}
    tokens, pairs = _seen(case, cached, new)
    heads = case["kv_heads"] * case["group"]
    return {"bytes": int(4 * new.sum() * heads * case["dim"] + 2 * tokens.sum() * case["kv_heads"] * _row_bytes(case)
                         + 4 * _pages(tokens, case["page"]).sum() + 8 * case["requests"]
                         + (16 * new.sum() if case["seen"] == "tree" else 0)),
            "flops": int(4 * case["dim"] * heads * pairs.sum())}


def _quantize(x, bits):
    """Codes (in 4 bits two a byte) and scale bytes of float32 rows, 32 values a block."""
    blocks = x.unflatten(-1, (x.shape[-1] // 32, 32))
    most = blocks.abs().amax(-1).view(torch.int32)
    # amax < 464 * 2^(scale - 127), 7 * 2^(scale - 127): what is above the largest code is nearer to it than to the next
    scale = ((most.long() + 0x180000 >> 23) - 8 if bits == 8 else (most.long() + 0x200000 >> 23) - 2).clamp(min=0)
    broken = most >= 0x7F800000
    y = torch.ldexp(blocks.abs(), (127 - scale).unsqueeze(-1)).masked_fill(broken.unsqueeze(-1), 0.0)
    byte = torch.where(broken, 255, scale).to(torch.uint8)
    if bits == 8:
        return torch.copysign(y.clamp(max=448.0), blocks).to(FLOAT8).view(x.shape), byte
    code = (y > 0.25).byte() + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0)
    code = torch.where(broken.unsqueeze(-1), 0, code + 8 * torch.signbit(blocks)).to(torch.uint8).reshape(x.shape)
    return code[..., 0::2] | code[..., 1::2] << 4, byte


def _values(codes, scales, bits):
    """float32 rows from the codes' bytes and scale bytes [..., dim / 32]."""
    if bits == 8:
        x = codes.view(FLOAT8).float().unflatten(-1, (scales.shape[-1], 32))
    else:
        level = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float32, device=codes.device)
        x = level[torch.stack([codes & 15, codes >> 4], -1).reshape(*scales.shape, 32).int()]
    e = scales.int() - 127
    half = torch.div(e, 2, rounding_mode="floor")                        # two factors: 2^-127 is not a normal number
    x = x * torch.exp2(half.float()).unsqueeze(-1) * torch.exp2((e - half).float()).unsqueeze(-1)
    return x.masked_fill((scales == 255).unsqueeze(-1), math.nan).flatten(-2)


def _made(gen, shape, dtype):
    """Rows as projections give them: normal, channels of different sizes."""
    x = torch.randn(shape, generator=gen, device=gen.device, dtype=torch.float32)
    return (x * torch.rand(shape[-1], generator=gen, device=gen.device).mul_(1.5).add_(0.25)).to(dtype)


def _made_cache(gen, case, pages, layers=1):
    """A cache full of rounded rows, as (codes, scales) with the layers in front."""
    shape = (layers * pages, case["kv_heads"], 2, case["page"])
    cache = torch.empty((*shape, case["dim"] * case["bits"] // 8), dtype=torch.uint8, device=gen.device)
    scales = torch.empty((*shape[:3], case["dim"] // 32, case["page"]), dtype=torch.uint8, device=gen.device)
    step = max(1, 200_000_000 // (case["kv_heads"] * 2 * case["page"] * case["dim"]))
    for p in range(0, len(cache), step):
        codes, s = _quantize(_made(gen, (len(cache[p:p + step]), *shape[1:], case["dim"]), torch.float32), case["bits"])
        cache[p:p + step], scales[p:p + step] = codes.view(torch.uint8), s.transpose(-1, -2)
    cache = cache.view(FLOAT8) if case["bits"] == 8 else cache
    return cache.view(layers, pages, *cache.shape[1:]), scales.view(layers, pages, *scales.shape[1:])


def _parents(rng, new, chains):
    """Trees as drafts grow: a node goes on from any node before it, rather from late ones; a prompt is a chain."""
    parents = [np.maximum(np.arange(n) * rng.random(n) ** 0.6, 0).astype(np.int64) for n in new]
    for b, p in enumerate(parents):
        p[:] = np.arange(len(p)) - 1 if b < chains else np.minimum(p, np.arange(len(p)) - 1)
    return parents


def _numbered(parents):
    """The four words of each node."""
    n = len(parents)
    size, depth, taken, number = [1] * n, [0] * n, [0] * (n + 1), [0] * n
    for i in range(n - 1, -1, -1):
        if parents[i] >= 0:
            size[parents[i]] += size[i]
    for i, p in enumerate(parents):
        depth[i] = depth[p] + 1 if p >= 0 else 0
        number[i] = taken[p] + (number[p] + 1 if p >= 0 else 0)          # (taken[-1]: the roots')
        taken[p] += size[i]
    least = np.minimum.accumulate(np.array(depth[::-1], np.int64))[::-1]
    return np.stack([number, size, depth, least], 1) if n else np.zeros((0, 4), np.int64)


def _draft(rng, parents, n):
    """Drafted tokens and the model's choices behind each node, which follow a path for some way. Kept rows do not
    lie on each other's places, so that a second pass finds what the first one found."""
    tokens, picked = rng.integers(0, 30_000, n), rng.integers(0, 30_000, n)
    path = [0]
    while True:
        follow = [c for c in range(path[-1] + 1, n) if parents[c] == path[-1]]
        more = path + [follow[int(rng.integers(len(follow)))]] if follow and rng.random() < 0.85 else None
        if more is None or any(k != i and k < len(more) for i, k in enumerate(more)):
            picked[path[-1]] = 30_001
            return tokens, picked
        tokens[[c for c in follow if c != more[-1]]] = 30_002              # the other branches drafted something else
        picked[path[-1]] = tokens[more[-1]]
        path = more


def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    dtype = DTYPES[case["dtype"]]
    put = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to(device=dev, dtype=t)
    if case["kind"] == "rows":
        n, heads, dim, page = case["tokens"], case["kv_heads"], case["dim"], case["page"]
        pages = _pages(n, page) + 3
        joint = _made(gen, (n, 4 * heads, dim), dtype)                   # queries, keys, values side by side
        # requests fill their pages token by token; the pages lie anywhere
        slots = (rng.permutation(pages)[:, None] * page + np.arange(page)[None, :]).reshape(-1)[:n].astype(np.int64)
        slots[rng.random(n) < case["skip"]] = -1
        return dict(kind="rows", dtype=dtype, keys=joint[:, 2 * heads:3 * heads], values=joint[:, 3 * heads:],
                    slots=put(slots, torch.int64), back=put(rng.permutation(slots), torch.int64),
                    cache=torch.zeros((pages, heads, 2, page, dim), dtype=torch.uint8, device=dev).view(FLOAT8),
                    scales=torch.zeros((pages, heads, 2, dim // 32, page), dtype=torch.uint8, device=dev))
    cached, new = _lengths(case)
    if case["kind"] == "tree":
        chains = int(case["prompts"] * case["requests"])
    order = rng.permutation(case["requests"])
    if case["kind"] != "tree":
        cached, new, chains = cached[order], new[order], 0
    parents = _parents(rng, new, chains)
    starts = np.concatenate([[0], np.cumsum(new)])
    if case["kind"] == "tree":
        return dict(kind="tree", parents=put(np.concatenate(parents), torch.int32), starts=put(starts, dtype),
                    kv_lens=put(cached + new, dtype), most_new=int(new.max()))
    page = case["page"]
    total = cached if case["kind"] == "attend" and case["seen"] == "all" else cached + new
    width = int(max(1, _pages(total, page).max()))
    keep = np.arange(width)[None, :] < _pages(total, page)[:, None]
    if case["kind"] == "attend" and case["window"]:                      # pages that no row can see were given back
        first = np.maximum(cached - case["window"] + 1, 0)
        keep &= (np.arange(width)[None, :] >= (first // page)[:, None]) | (np.arange(width) * page < case["sinks"])
    used = int(keep.sum())
    pool = rng.permutation(used + 5)
    table = np.full((case["requests"], width), -1, dtype=np.int64)
    table[keep] = pool[:used]
    common = dict(kind=case["kind"], table=put(table, torch.int32), starts=put(starts, torch.int32),
                  kv_lens=put(total, torch.int32), most_new=int(new.max()), bits=case["bits"])
    if case["kind"] == "keep":
        drafts = [_draft(rng, p, len(p)) for p in parents]
        cache, scales = _made_cache(gen, case, len(pool), case["layers"])
        return dict(common, cache=cache, scales=scales, parents=put(np.concatenate(parents), torch.int32),
                    tokens=put(np.concatenate([d[0] for d in drafts]), dtype),
                    picked=put(np.concatenate([d[1] for d in drafts]), dtype))
    cache, scales = _made_cache(gen, case, len(pool))
    nodes = np.concatenate([_numbered(p.tolist()) for p in parents]) if case["seen"] == "tree" else None
    return dict(common, dtype=dtype, cache=cache[0], scales=scales[0], seen=case["seen"],
                query=2.0 * _made(gen, (int(new.sum()), case["kv_heads"] * case["group"], case["dim"]), dtype),
                nodes=None if nodes is None else put(nodes, torch.int32), scale=case["dim"] ** -0.5,
                window=case["window"], sinks=case["sinks"], most_kv=max(1, int(total.max())))


def _padded(x, starts, most, fill):
    """x [tokens, ...] as [requests, most, ...], and which of those are there."""
    i = torch.arange(most, device=x.device)
    there = i < (starts[1:] - starts[:-1])[:, None]
    rows = (starts[:-1, None] + i).long().clamp(max=max(len(x) - 1, 0))
    shape = (*there.shape, *[1] * (x.dim() - 1))
    return torch.where(there.view(shape), x[rows], fill), there, rows


def _ancestors(parents):
    """float [requests, nodes, nodes]: whether the second is the first or above it, for padded parents."""
    n = parents.shape[1]
    above = torch.eye(n + 1, device=parents.device, dtype=torch.bool).expand(len(parents), -1, -1).clone()
    above[:, :, n] = False                                               # the last row is nobody, who is above the roots
    jump = torch.cat([torch.where(parents < 0, n, parents), torch.full_like(parents[:, :1], n)], 1).long()
    for _ in range(max(1, (n - 1).bit_length())):                        # twice as many generations a turn
        above = above | above.gather(1, jump[:, :, None].expand(-1, -1, n + 1))
        jump = jump.gather(1, jump)
    return above[:, :n, :n]


def _tree(parents, starts, kv_lens, most):
    p, there, rows = _padded(parents, starts, most, -1)
    n = p.shape[1]
    above = _ancestors(p).float() * there[:, :, None]
    size = above.sum(1)                                                  # whole numbers far below 2^24 throughout
    depth = above.sum(2) - 1
    i = torch.arange(n, device=p.device)
    same = (p[:, :, None] == p[:, None, :]) & (i[None, :] < i[:, None])
    before = torch.matmul(same.float(), size[:, :, None])                # of the earlier children of the same parent
    number = torch.matmul(above, before)[:, :, 0] + depth
    least = torch.where(there, depth, 3e9).flip(1).cummin(1)[0].flip(1)
    nodes = torch.stack([number, size, depth, least], 2)[there].int()
    first = (kv_lens - (starts[1:] - starts[:-1]))[:, None]
    return [nodes, (first + depth.long())[there].int()]


def _keep(cache, scales, table, starts, kv_lens, parents, tokens, picked, most):
    """The path from node 0 on: a node is on it if it, and all above it but node 0, is the first child whose token was picked."""
    page = scales.shape[-1]
    p, there, rows = _padded(parents, starts, most, -1)
    above = _ancestors(p)
    asked = picked[rows].gather(1, p.clamp(min=0).long())
    right = there & (p >= 0) & (tokens[rows] == asked)
    i = torch.arange(most, device=p.device)
    earlier = (p[:, :, None] == p[:, None, :]) & (i[None, :] < i[:, None]) & right[:, None, :]
    chosen = (right & ~earlier.any(2)) | (i == 0)
    on = there & (above <= chosen[:, None, :]).all(2) & above[:, :, 0]
    counts = on.sum(1)
    place = on.cumsum(1) - 1
    path = torch.full_like(rows, -1)
    b, node = on.nonzero(as_tuple=True)
    path[b, place[b, node]] = node
    last = path.gather(1, (counts - 1).clamp(min=0)[:, None])
    follow = torch.where(counts > 0, picked[rows].gather(1, last.clamp(min=0))[:, 0], -1)
    first = (kv_lens - (starts[1:] - starts[:-1])).long()
    src, dst = first[b] + node, first[b] + place[b, node]
    at, off, to, to_off = table[b, src // page].long(), src % page, table[b, dst // page].long(), dst % page
    raw = cache.view(torch.uint8)
    raw[:, to, :, :, to_off] = raw[:, at, :, :, off]
    turned = scales.transpose(-1, -2)
    turned[:, to, :, :, to_off] = turned[:, at, :, :, off]
    return [counts.int(), path[there].int(), follow, raw, scales]


def _rows(cache, scales, slots, keys, values, back, dtype):
    page, raw = cache.shape[3], cache.view(torch.uint8)
    keep = (slots >= 0).nonzero()[:, 0]
    codes, s = _quantize(torch.stack([keys[keep].float(), values[keep].float()], 2), 8)
    at, off = slots[keep] // page, slots[keep] % page
    raw[at, :, :, off] = codes.view(torch.uint8)
    scales.transpose(-1, -2)[at, :, :, off] = s
    seat = back.clamp(min=0)
    at, off = seat // page, seat % page
    x = _values(raw[at, :, :, off], scales.transpose(-1, -2)[at, :, :, off], 8)
    x = torch.where((back >= 0)[:, None, None, None], x, 0.0).to(dtype)
    return [x[:, :, 0].contiguous(), x[:, :, 1].contiguous()]


def _attend(query, cache, scales, table, starts, kv_lens, scale, window, sinks, most_new, most_kv, seen, nodes, bits):
    """Padded: every request has most_new queries and most_kv tokens, those that it lacks are masked."""
    dev, (n, heads, dim), page, raw = query.device, query.shape, cache.shape[3], cache.view(torch.uint8)
    kv_heads = cache.shape[1]
    token = torch.arange(most_kv, device=dev)
    at = table[:, token // page].long()                                             # [requests, tokens]
    there = (at >= 0) & (token < kv_lens[:, None])
    at = at.clamp(min=0)
    off = (token % page).expand_as(at)
    q, mine, row = _padded(query, starts, most_new, 0.0)
    q = q.float()                                                                   # [requests, queries, heads, dim]
    first = (kv_lens - (starts[1:] - starts[:-1])).long()[:, None]
    i = torch.arange(most_new, device=dev)
    pos, place, sees = first + i, token.expand_as(at), there[:, None, :]
    if seen == "causal":
        sees = sees & (token <= pos[:, :, None])
    if seen == "tree":
        node, _, _ = _padded(nodes, starts, most_new, 0)
        number, size, depth = node[..., 0], node[..., 1], node[..., 2].long()
        above = ((number[:, :, None] >= number[:, None, :])
                 & (number[:, :, None] < (number + size)[:, None, :]))              # [requests, queries, nodes]
        j = (token - first).clamp(0, most_new - 1)
        fresh = token >= first
        sees = sees & (~fresh[:, None, :] | above.gather(2, j[:, None, :].expand(-1, most_new, -1)))
        pos, place = first + depth, torch.where(fresh, first + depth.gather(1, j), token)
    if window:
        sees = sees & ((place[:, None, :] > pos[:, :, None] - window) | (place < sinks)[:, None, :])
    q = q.reshape(*q.shape[:2], kv_heads, -1, dim).permute(0, 2, 3, 1, 4).flatten(2, 3).contiguous()
    k = _values(raw[at, :, 0, off], scales[at, :, 0, :, off], bits).permute(0, 2, 3, 1).contiguous()
    s = torch.matmul(q, k).mul_(scale).unflatten(2, (-1, most_new))
    del k
    s.masked_fill_(~sees[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = s.sum(-1, keepdim=True)
    v = _values(raw[at, :, 1, off], scales[at, :, 1, :, off], bits).masked_fill_(~there[:, :, None, None], 0.0)
    out = torch.matmul(s.flatten(2, 3), v.transpose(1, 2).contiguous()).unflatten(2, (-1, most_new))
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).flatten(2, 3)
    answer = torch.zeros((n + 1, heads, dim), dtype=torch.float32, device=dev)
    answer[torch.where(mine, row, n)] = out                                         # what no request has goes to row n
    return answer[:n].to(query.dtype)


def run(state):
    s = state
    if own:
        import shmtensor_amd
        capi = shmtensor_amd.ShmTensorLib
        if s["kind"] == "tree":
            return capi.page_tree(s["parents"], s["starts"], s["kv_lens"])
        if s["kind"] == "keep":
            return [*capi.page_keep(s["cache"], s["scales"], s["table"], s["starts"], s["kv_lens"], s["parents"],
                                    s["tokens"], s["picked"]), s["cache"].view(torch.uint8), s["scales"]]
        if s["kind"] == "rows":
            capi.page_set(s["cache"], s["scales"], s["slots"], s["keys"], s["values"])
            return capi.page_fetch(s["cache"], s["scales"], s["back"], s["dtype"])
        return capi.page_attention(s["query"], s["cache"], s["scales"], s["table"], s["starts"], s["kv_lens"],
                                   s["scale"], window=s["window"], sinks=s["sinks"], max_query_len=s["most_new"],
                                   tree=s["nodes"], causal=s["seen"] != "all")
    if s["kind"] == "tree":
        return _tree(s["parents"], s["starts"], s["kv_lens"], s["most_new"])
    if s["kind"] == "keep":
        return _keep(s["cache"], s["scales"], s["table"], s["starts"], s["kv_lens"], s["parents"], s["tokens"],
                     s["picked"], s["most_new"])
    if s["kind"] == "rows":
        return _rows(s["cache"], s["scales"], s["slots"], s["keys"], s["values"], s["back"], s["dtype"])
    return _attend(s["query"], s["cache"], s["scales"], s["table"], s["starts"], s["kv_lens"], s["scale"],
                   s["window"], s["sinks"], s["most_new"], s["most_kv"], s["seen"], s["nodes"], s["bits"])


def _exact_row(codes, scales, bits):
    """float64 rows from the codes' bytes [n, ...] and scale bytes [dim / 32, n]."""
    c = codes.long() if bits == 8 else torch.stack([codes & 15, codes >> 4], -1).flatten(1).long()
    mantissa, bias = (3, 7) if bits == 8 else (1, 1)
    e, m = (c >> mantissa) & (15 if bits == 8 else 3), (c & (1 << mantissa) - 1).double() / (1 << mantissa)
    size = torch.where(e > 0, (1.0 + m) * torch.exp2((e - bias).double()), m * 2.0 ** (1 - bias))
    size = torch.where(c >> (bits - 1) > 0, -size, size)
    return size * torch.exp2(scales.t().double() - 127).repeat_interleave(32, 1)


def _exact_rounded(x):
    """float64 values that rows are rounded to in 8 bits: steps of 2^-3 of a value's power of two, or 2^-9, up to 448."""
    x = x.double().unflatten(-1, (-1, 32))
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))                   # the largest is m 2^e, m in [0.5, 1)
    power = torch.exp2((e - 9 + (m >= 0.90625).int()).clamp(min=-127).double())
    y = (x / power).abs()
    step = torch.exp2((torch.frexp(y)[1] - 1).clamp(min=-6).double() - 3)
    return (torch.sign(x) * torch.clamp(torch.round(y / step) * step, max=448.0) * power).flatten(-2)


def _exact_path(parents, tokens, picked):
    path = [0] if parents else []
    for c in range(1, len(parents)):                                     # children come behind their parents
        if parents[c] == path[-1] and tokens[c] == picked[path[-1]]:
            path.append(c)
    return path


def _forest(parents):
    """The four words of each node, by walking down from the roots."""
    n = len(parents)
    children = {p: [c for c in range(n) if parents[c] == p] for p in set(parents)}
    words, todo, last = np.zeros((n, 4), np.int32), [(r, 0) for r in reversed(children.get(-1, []))], 0
    while todo:
        i, depth = todo.pop()
        words[i, 0], words[i, 2], last = last, depth, last + 1
        todo += [(c, depth + 1) for c in reversed(children.get(i, []))]
    above = [{i} for i in range(n)]
    for i, p in enumerate(parents):
        above[i] |= above[p] if p >= 0 else set()
        for a in above[i]:
            words[a, 1] += 1
    words[:, 3] = [words[i:, 2].min() for i in range(n)]
    return words


def exact(case, seed):
    if case["kind"] == "attend" and not torch.cuda.is_available() and work(case)["flops"] > 2e10:
        return None
    s = prepare(case, seed)
    if case["kind"] == "rows":
        # the rows that were set, by slot; every slot that is read was set
        seat = torch.zeros(s["cache"].shape[0] * case["page"], dtype=torch.int64, device=s["slots"].device)
        put = s["slots"] >= 0
        seat[s["slots"][put]] = torch.arange(case["tokens"], device=seat.device)[put]
        source = seat[s["back"].clamp(min=0)]
        return [torch.where((s["back"] >= 0)[:, None, None], _exact_rounded(x[source]), 0.0)
                for x in (s["keys"], s["values"])]
    starts, lens = s["starts"].tolist(), s["kv_lens"].tolist()
    if case["kind"] == "tree":
        parents = s["parents"].tolist()
        words = [_forest(parents[lo:hi]) for lo, hi in zip(starts, starts[1:])]
        places = [w[:, 2] + length - len(w) for w, length in zip(words, lens)]
        return [np.concatenate(words), np.concatenate(places).astype(np.int32)]
    if case["kind"] == "keep":
        parents, tokens, picked, table = (s[k].tolist() for k in ("parents", "tokens", "picked", "table"))
        counts, paths, follow, page = [], [], [], case["page"]
        cache, scales = s["cache"].view(torch.uint8), s["scales"]
        src, dst = [], []
        for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
            path = _exact_path(parents[lo:hi], tokens[lo:hi], picked[lo:hi])
            first = lens[b] - (hi - lo)
            src += [table[b][(first + node) // page] * page + (first + node) % page for node in path]
            dst += [table[b][(first + k) // page] * page + (first + k) % page for k in range(len(path))]
            counts.append(len(path))
            paths += path + [-1] * (hi - lo - len(path))
            follow.append(picked[lo + path[-1]] if path else -1)
        src, dst = (torch.tensor(x, device=cache.device) for x in (src, dst))
        for held, codes in ((cache, True), (scales, False)):             # places of a page side by side with the pages
            x = (held if codes else held.transpose(-1, -2)).permute(1, 4, 0, 2, 3, 5)
            flat = x.reshape(-1, *x.shape[2:])
            flat[dst] = flat[src]
            x.copy_(flat.view(x.shape))
        return [np.array(counts, np.int32), np.array(paths, np.int32), np.array(follow), cache, scales]
    raw = s["cache"].view(torch.uint8)
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=s["query"].device)
    group, page, bits, window, sinks = case["group"], case["page"], case["bits"], case["window"], case["sinks"]
    for b, length in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        if lo == hi or length == 0:
            continue
        j = torch.arange(length, device=out.device)
        where = s["table"][b].long()[j // page]
        first = length - (hi - lo)
        place, pos = j, torch.arange(first, length, device=out.device)[:, None]
        hidden = torch.zeros((hi - lo, length), dtype=torch.bool, device=out.device)
        if case["seen"] == "tree":
            number, size, depth = s["nodes"][lo:hi, :3].long().unbind(1)
            gap = number[:, None] - number[None, :]
            hidden[:, first:] = (gap < 0) | (gap >= size[None, :])
            place, pos = torch.cat([j[:first], first + depth]), first + depth[:, None]
        elif case["seen"] == "causal":
            hidden |= j[None, :] > pos
        if window:
            hidden |= (place[None, :] <= pos - window) & (place[None, :] >= sinks)
        hidden |= (where < 0)[None, :]
        at = (~hidden).any(0).nonzero()[:, 0]
        where, off, hidden = where[at], at % page, hidden[:, at]
        for h in range(case["kv_heads"]):
            k, v = (_exact_row(raw[where, h, i, off], s["scales"][where, h, i, :, off].t(), bits) for i in (0, 1))
            for g in range(h * group, (h + 1) * group):
                score = s["query"][lo:hi, g].double() @ k.t() * s["scale"]
                out[lo:hi, g] = torch.softmax(score.masked_fill_(hidden, -math.inf), -1) @ v
    return out
