"""Performance cases of the paged key/value cache held in 4 bits: what a program that serves a language model asks of it.

Such a program keeps the keys and values of its running requests in pages of `page` tokens in HBM. A step gets the
requests' lengths (how many tokens are cached, how many are new), assigns pages and slots to the new tokens (`plan`),
writes their keys and values to the slots and reads some of them back (`rows`), and lets the new tokens' queries attend
to everything that their request holds, or to a window of it and a few first tokens (`attend`).

A cached row of `dim` values is held as 4-bit floats (sign, 2 bits of exponent, 1 of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4,
6) with one power of two for every 32 values:

    cache   uint8 [pages, kv_heads, 2, page, dim / 2]    keys at 0, values at 1; the even dimension in the low bits
    scales  uint8 [pages, kv_heads, 2, dim / 32, page]   2^(byte - 127); 255 stands for "not a number"
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "i32": torch.int32, "i64": torch.int64}
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # A decode step of a handful of requests: latency only.
        dict(name="plan_few", kind="plan", requests=7, cached_lo=10, cached_hi=2000, new_lo=1, new_hi=1, page=16,
             dtype="i32"),
        # A decode step of a full batch, one to four tokens a request (some are speculated).
        dict(name="plan_batch", kind="plan", requests=1024, cached_lo=1, cached_hi=16000, new_lo=1, new_hi=4, page=16,
             dtype="i32"),
        # Prompts of a whole queue: hundreds of thousands of tokens at once.
        dict(name="plan_prompts", kind="plan", requests=301, cached_lo=1, cached_hi=4000, new_lo=33, new_hi=8000,
             page=64, dtype="i64"),
        # The rows of one decode step.
        dict(name="rows_decode", kind="rows", tokens=61, kv_heads=8, dim=128, page=16, skip=0.05, dtype="bf16"),
        # Ragged chunk of prompts, narrow heads.
        dict(name="rows_chunk", kind="rows", tokens=5003, kv_heads=4, dim=64, page=32, skip=0.01, dtype="f16"),
        # Long prompts: the rows of 64 K tokens, slices of a joint projection.
        dict(name="rows_prompts", kind="rows", tokens=65_536, kv_heads=8, dim=128, page=64, skip=0.0, dtype="bf16"),
        # One user, a few hundred tokens: latency only.
        dict(name="attend_one", kind="attend", requests=1, cached_lo=700, cached_hi=700, new_lo=1, new_hi=1,
             kv_heads=8, group=4, dim=128, page=16, window=0, sinks=0, dtype="bf16"),
        # A decode step of a full batch of ragged requests.
        dict(name="attend_batch", kind="attend", requests=64, cached_lo=1000, cached_hi=16_000, new_lo=1, new_hi=1,
             kv_heads=8, group=4, dim=128, page=16, window=0, sinks=0, dtype="bf16"),
        # One long document, a few speculated tokens: the work has to be split over the cache.
        dict(name="attend_long", kind="attend", requests=1, cached_lo=130_001, cached_hi=130_001, new_lo=3, new_hi=3,
             kv_heads=8, group=5, dim=128, page=32, window=0, sinks=0, dtype="f16"),
        # Two whole prompts.
        dict(name="attend_prompts", kind="attend", requests=2, cached_lo=0, cached_hi=0, new_lo=8000, new_hi=8192,
             kv_heads=8, group=4, dim=128, page=64, window=0, sinks=0, dtype="bf16"),
        # Decode of long requests that keep a window and a few first tokens; pages in between were given back.
        dict(name="attend_window_decode", kind="attend", requests=96, cached_lo=3000, cached_hi=30_000, new_lo=1,
             new_hi=1, kv_heads=8, group=8, dim=64, page=16, window=4000, sinks=5, dtype="f16"),
        # Chunks of prompts with a window, wide heads, requests of all lengths.
        dict(name="attend_window_chunks", kind="attend", requests=5, cached_lo=100, cached_hi=9000, new_lo=17,
             new_hi=2000, kv_heads=2, group=8, dim=256, page=32, window=1000, sinks=4, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    kind = rng.choice(["plan", "rows", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        n = _log_int(rng, 1, 2000)
        new_hi = _log_int(rng, 1, max(1, min(8000, 500_000 // n)))
        cached_hi = _log_int(rng, 1, 16_000)
        return dict(kind=kind, requests=n, cached_lo=rng.choice([0, 1, min(cached_hi, 100)]), cached_hi=cached_hi,
                    new_lo=rng.choice([0, 1, new_hi]), new_hi=new_hi, page=page, dtype=rng.choice(["i32", "i64"]))
    if kind == "rows":
        return dict(kind=kind, tokens=_log_int(rng, 1, 40_000), kv_heads=rng.choice([1, 2, 3, 5, 8]),
                    dim=rng.choice([64, 128, 256]) if rng.random() < 0.5 else 128, page=page,
                    skip=rng.choice([0.0, 0.02, 0.3]), dtype=rng.choice(["bf16", "f16", "f32"]))
    kv_heads, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), rng.choice([64, 128, 256])
    mode = rng.choice(["decode", "decode", "few", "prompts"])
    n = _log_int(rng, 1, 128 if mode == "decode" else 32 if mode == "few" else 6)
    wide = n * kv_heads * dim
    cached_hi = _log_int(rng, 1, max(1, min(100_000, 400_000_000 // wide)))
    new_hi = 1 if mode == "decode" else rng.randint(2, 9) if mode == "few" else _log_int(rng, 10, 4000)
    heads = n * kv_heads * group * new_hi
    cached_hi = max(1, min(cached_hi, 1_500_000_000 // heads - new_hi))
    new_hi = min(new_hi, max(1, 1_500_000_000 // (n * kv_heads * group * (cached_hi + new_hi))))
    window = rng.choice([0, 0, _log_int(rng, 1, 8000)])
    return dict(kind=kind, requests=n, cached_lo=rng.choice([0, min(cached_hi, 20), max(1, cached_hi // 8)]),
                cached_hi=cached_hi, new_lo=rng.choice([1, max(1, new_hi // 4)]), new_hi=new_hi, kv_heads=kv_heads,
                group=group, dim=dim, page=page, window=window, sinks=rng.choice([0, 1, 4, 37]) if window else 0,
                dtype=rng.choice(["bf16", "f16"]))


def _lengths(case):
    """(cached, new) of each request: spread over their ranges (by their logarithm), the same for every seed."""
    def spread(lo, hi, step):
        at = np.mod((np.arange(case["requests"]) + 0.5) * step, 1.0)
        return np.rint((lo + 1) * ((hi + 1) / (lo + 1)) ** at - 1).astype(np.int64)
    return (spread(case["cached_lo"], case["cached_hi"], 0.6180339887),
            spread(case["new_lo"], case["new_hi"], 0.7548776662))


def _pages(tokens, page):
    return -(-tokens // page)


def _seen(case, cached, new):
    """(tokens that some row of the request sees, pairs of a row and a token that it sees), per request."""
    total, w, s = cached + new, case["window"], case["sinks"]
    if not w:
        return total, new * cached + new * (new + 1) // 2
    first = np.maximum(cached - w + 1, 0)                     # the first row's window begins here
    tokens = np.minimum(total, s) + total - np.maximum(first, np.minimum(total, s))
    # a row at position p sees min(p + 1, w) tokens of its window and the sinks in front of it
    def upto(p):                                              # rows 0 .. p - 1
        inside = np.minimum(p, w)
        pairs = inside * (inside + 1) // 2 + (p - inside) * w
        x = np.maximum(p - w, 0)                              # rows whose window begins after token 0: at 1 .. x
        low = np.minimum(x, s)
        return pairs + low * (low + 1) // 2 + (x - low) * s
    return np.where(new > 0, tokens, 0), upto(total) - upto(cached)


def work(case):
    """The bytes and the operations of one pass that nothing can do without."""
    if case["kind"] == "rows":
        values = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * (values * size + values // 2 + values // 32 + 8 * case["tokens"]), "flops": 2 * values}
    cached, new = _lengths(case)
    if case["kind"] == "plan":
        grown = int((_pages(cached + new, case["page"]) - _pages(cached, case["page"])).sum())
        size = 4 if case["dtype"] == "i32" else 8
        n, tokens = case["requests"], int(new.sum())
        return {"bytes": 2 * n * size + 4 * n + 8 * grown + 4 * (2 * n + 1) + 12 * tokens + 16, "flops": 2 * tokens + n}
    tokens, pairs = _seen(case, cached, new)
    heads = case["kv_heads"] * case["group"]
    row = case["dim"] // 2 + case["dim"] // 32
    return {"bytes": int(4 * new.sum() * heads * case["dim"] + 2 * tokens.sum() * case["kv_heads"] * row
                         + 4 * _pages(tokens, case["page"]).sum() + 8 * case["requests"]),
            "flops": int(4 * case["dim"] * heads * pairs.sum())}


def _quantize(x):
    """4-bit codes (two a byte) and scale bytes of float32 rows, 32 values a block."""
    blocks = x.unflatten(-1, (x.shape[-1] // 32, 32))
    bits = blocks.abs().amax(-1).view(torch.int32)
    scale = (((bits.long() + 0x200000) >> 23) - 2).clamp(min=0)          # amax < 7 * 2^(scale - 127)
    broken = bits >= 0x7F800000
    y = torch.ldexp(blocks.abs(), (127 - scale).unsqueeze(-1))
    code = (y > 0.25).byte() + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0)
    code = torch.where(broken.unsqueeze(-1), 0, code + 8 * torch.signbit(blocks)).to(torch.uint8)
    code = code.reshape(x.shape)
    return code[..., 0::2] | code[..., 1::2] << 4, torch.where(broken, 255, scale).to(torch.uint8)


def _values(codes, scales):
    """float32 rows from codes [..., dim / 2] and scale bytes [..., dim / 32]."""
    level = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float32, device=codes.device)
    code = torch.stack([codes & 15, codes >> 4], -1).reshape(*scales.shape, 32)
    e = scales.int() - 127
    half = torch.div(e, 2, rounding_mode="floor")                        # two factors: 2^-127 is not a normal number
    x = level[code.int()] * torch.exp2(half.float()).unsqueeze(-1) * torch.exp2((e - half).float()).unsqueeze(-1)
    return x.masked_fill((scales == 255).unsqueeze(-1), math.nan).flatten(-2)


def _made(gen, shape, dtype):
    """Rows as projections give them: normal, channels of different sizes."""
    x = torch.randn(shape, generator=gen, device=gen.device, dtype=torch.float32)
    return (x * torch.rand(shape[-1], generator=gen, device=gen.device).mul_(1.5).add_(0.25)).to(dtype)


def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    dtype, page = DTYPES[case["dtype"]], case["page"]
    put = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to(device=dev, dtype=t)
    if case["kind"] == "rows":
        n, heads, dim = case["tokens"], case["kv_heads"], case["dim"]
        pages = _pages(n, page) + 3
        joint = _made(gen, (n, 4 * heads, dim), dtype)                   # queries, keys, values side by side
        # requests fill their pages token by token; the pages lie anywhere
        slots = (rng.permutation(pages)[:, None] * page + np.arange(page)[None, :]).reshape(-1)[:n].astype(np.int64)
        slots[rng.random(n) < case["skip"]] = -1
        return dict(kind="rows", dtype=dtype, keys=joint[:, 2 * heads:3 * heads], values=joint[:, 3 * heads:],
                    slots=put(slots, torch.int64), back=put(rng.permutation(slots), torch.int64),
                    cache=torch.zeros((pages, heads, 2, page, dim // 2), dtype=torch.uint8, device=dev),
                    scales=torch.zeros((pages, heads, 2, dim // 32, page), dtype=torch.uint8, device=dev))
    cached, new = _lengths(case)
    order = rng.permutation(case["requests"])
    cached, new = cached[order], new[order]
    held = cached if case["kind"] == "plan" else cached + new
    total = cached + new
    width = int(max(1, _pages(total, page).max()))
    keep = np.arange(width)[None, :] < _pages(held, page)[:, None]
    if case["kind"] == "attend" and case["window"]:                      # pages that no row can see were given back
        first = np.maximum(cached - case["window"] + 1, 0)
        keep &= (np.arange(width)[None, :] >= (first // page)[:, None]) | (np.arange(width) * page < case["sinks"])
    used = int(keep.sum())
    grown = int((_pages(total, page) - _pages(held, page)).sum())
    pool = rng.permutation(used + grown + 5)
    table = np.full((case["requests"], width), -1, dtype=np.int64)
    table[keep] = pool[:used]
    if case["kind"] == "plan":
        return dict(kind="plan", cached=put(cached, dtype), new=put(new, dtype), table=put(table, torch.int32),
                    free=put(pool[used:], torch.int32), page=page, tokens=int(new.sum()))
    heads, dim, pages = case["kv_heads"], case["dim"], len(pool)
    cache = torch.empty((pages, heads, 2, page, dim // 2), dtype=torch.uint8, device=dev)
    scales = torch.empty((pages, heads, 2, dim // 32, page), dtype=torch.uint8, device=dev)
    step = max(1, 400_000_000 // (heads * 2 * page * dim))
    for p in range(0, pages, step):
        codes, s = _quantize(_made(gen, (len(cache[p:p + step]), heads, 2, page, dim), torch.float32))
        cache[p:p + step], scales[p:p + step] = codes, s.transpose(-1, -2)
    starts = np.concatenate([[0], np.cumsum(new)])
    return dict(kind="attend", dtype=dtype, cache=cache, scales=scales, table=put(table, torch.int32),
                query=2.0 * _made(gen, (int(new.sum()), heads * case["group"], dim), dtype),
                starts=put(starts, torch.int32), kv_lens=put(total, torch.int32), scale=dim ** -0.5,
                window=case["window"], sinks=case["sinks"], most_new=int(new.max()), most_kv=int(total.max()))


def _plan(cached, new, table, free, page, tokens):
    total = cached + new
    have, need = (cached + page - 1) // page, (total + page - 1) // page
    before = torch.cumsum(need - have, 0) - (need - have)
    column = torch.arange(table.shape[1], device=table.device)[None, :]
    fresh = (column >= have[:, None]) & (column < need[:, None])
    table.copy_(torch.where(fresh, free[(before[:, None] + column - have[:, None]).clamp(0, free.numel() - 1)], table))
    ends = torch.cumsum(new, 0)
    at = torch.arange(tokens, device=table.device)
    row = torch.searchsorted(ends, at, right=True)
    pos = cached[row] + at - (ends - new)[row]
    slots = table[row, pos // page].long() * page + pos % page
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    return [starts.int(), total.int(), pos.int(), slots, torch.stack([ends[-1], (need - have).sum()]).long(), table]


def _rows(cache, scales, slots, keys, values, back, dtype):
    page = cache.shape[3]
    keep = (slots >= 0).nonzero()[:, 0]
    codes, s = _quantize(torch.stack([keys[keep].float(), values[keep].float()], 2))
    at, off = slots[keep] // page, slots[keep] % page
    cache[at, :, :, off] = codes
    scales.transpose(-1, -2)[at, :, :, off] = s
    seat = back.clamp(min=0)
    at, off = seat // page, seat % page
    x = _values(cache[at, :, :, off], scales.transpose(-1, -2)[at, :, :, off])
    x = torch.where((back >= 0)[:, None, None, None], x, 0.0).to(dtype)
    return [x[:, :, 0].contiguous(), x[:, :, 1].contiguous()]


def _attend(query, cache, scales, table, starts, kv_lens, scale, window, sinks, most_new, most_kv):
    """Padded: every request has most_new queries and most_kv tokens, those that it lacks are masked."""
    dev, (n, heads, dim), page = query.device, query.shape, cache.shape[3]
    kv_heads = cache.shape[1]
    token = torch.arange(most_kv, device=dev)
    at = table[:, token // page].long()                                             # [requests, tokens]
    there = (at >= 0) & (token < kv_lens[:, None])
    at = at.clamp(min=0)
    off = (token % page).expand_as(at)
    i = torch.arange(most_new, device=dev)
    news = (starts[1:] - starts[:-1]).long()
    row = starts[:-1, None].long() + i
    mine = i < news[:, None]
    pos = (kv_lens.long() - news)[:, None] + i                                      # [requests, queries]
    sees = there[:, None, :] & (token <= pos[:, :, None])
    if window:
        sees = sees & ((token > pos[:, :, None] - window) | (token < sinks))
    q = query[row.clamp(max=max(n - 1, 0))].float()                                 # [requests, queries, heads, dim]
    q = q.reshape(*q.shape[:2], kv_heads, -1, dim).permute(0, 2, 3, 1, 4).flatten(2, 3).contiguous()
    k = _values(cache[at, :, 0, off], scales[at, :, 0, :, off]).permute(0, 2, 3, 1).contiguous()
    s = torch.matmul(q, k).mul_(scale).unflatten(2, (-1, most_new))
    del k
    hidden = ~sees[:, None, None]
    s.masked_fill_(hidden, -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = s.sum(-1, keepdim=True)
    v = _values(cache[at, :, 1, off], scales[at, :, 1, :, off]).masked_fill_(~there[:, :, None, None], 0.0)
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
        if s["kind"] == "plan":
            return [*capi.page_plan(s["cached"], s["new"], s["table"], s["free"], s["page"], s["tokens"]), s["table"]]
        if s["kind"] == "rows":
            capi.page_set(s["cache"], s["scales"], s["slots"], s["keys"], s["values"])
            return capi.page_fetch(s["cache"], s["scales"], s["back"], s["dtype"])
        return capi.page_attention(s["query"], s["cache"], s["scales"], s["table"], s["starts"], s["kv_lens"],
                                   s["scale"], window=s["window"], sinks=s["sinks"], max_query_len=s["most_new"])
    if s["kind"] == "plan":
        return _plan(s["cached"], s["new"], s["table"], s["free"], s["page"], s["tokens"])
    if s["kind"] == "rows":
        return _rows(s["cache"], s["scales"], s["slots"], s["keys"], s["values"], s["back"], s["dtype"])
    return _attend(s["query"], s["cache"], s["scales"], s["table"], s["starts"], s["kv_lens"], s["scale"],
                   s["window"], s["sinks"], s["most_new"], s["most_kv"])


def _exact_row(codes, scales):
    """float64 rows from codes [n, dim / 2] and scale bytes [dim / 32, n]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(1).long()
    e, m = (c >> 1) & 3, c & 1
    size = torch.where(e > 0, (1.0 + 0.5 * m.double()) * torch.exp2((e - 1).double()), 0.5 * m.double())
    size = torch.where(c > 7, -size, size)
    return size * torch.exp2(scales.t().double() - 127).repeat_interleave(32, 1)


def _exact_rounded(x):
    """float64 values that rows are rounded to: a step of 0.5, 1 or 2 times the block's power of two, at most 6 times."""
    x = x.double().unflatten(-1, (-1, 32))
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))
    power = torch.exp2((e - 3 + (m >= 0.875).int()).clamp(min=-127).double())
    y = (x / power).abs()
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0)).double()
    return (torch.sign(x) * torch.clamp(torch.round(y / step) * step, max=6.0) * power).flatten(-2)


def exact(case, seed):
    if case["kind"] == "attend" and not torch.cuda.is_available() and work(case)["flops"] > 2e10:
        return None
    s = prepare(case, seed)
    if case["kind"] == "plan":
        cached, new, free = s["cached"].tolist(), s["new"].tolist(), s["free"].tolist()
        table, page = s["table"].tolist(), case["page"]
        starts, lens, pos, slots, taken = [0], [], [], [], 0
        for b, (c, n) in enumerate(zip(cached, new)):
            for p in range(-(-c // page), -(-(c + n) // page)):
                table[b][p] = free[taken]
                taken += 1
            starts.append(starts[-1] + n)
            lens.append(c + n)
            pos += range(c, c + n)
            slots += [table[b][p // page] * page + p % page for p in range(c, c + n)]
        return [np.array(starts, np.int32), np.array(lens, np.int32), np.array(pos, np.int32), np.array(slots, np.int64),
                np.array([starts[-1], taken], np.int64), np.array(table, np.int32)]
    if case["kind"] == "rows":
        # the rows that were set, by slot; every slot that is read was set
        seat = torch.zeros(s["cache"].shape[0] * case["page"], dtype=torch.int64, device=s["slots"].device)
        put = s["slots"] >= 0
        seat[s["slots"][put]] = torch.arange(case["tokens"], device=seat.device)[put]
        source = seat[s["back"].clamp(min=0)]
        return [torch.where((s["back"] >= 0)[:, None, None], _exact_rounded(x[source]), 0.0)
                for x in (s["keys"], s["values"])]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=s["query"].device)
    starts, lens, group, page = s["starts"].tolist(), s["kv_lens"].tolist(), case["group"], case["page"]
    for b, length in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        if lo == hi:
            continue
        first = length - (hi - lo)
        seen = torch.zeros(length, dtype=torch.bool, device=out.device)
        seen[max(0, first - case["window"] + 1) if case["window"] else 0:] = True
        seen[:case["sinks"]] = True
        at = seen.nonzero()[:, 0]
        where, off = s["table"][b].long()[at // page], at % page
        pos = torch.arange(first, length, device=out.device)[:, None]
        hidden = at[None, :] > pos
        if case["window"]:
            hidden |= (at[None, :] <= pos - case["window"]) & (at[None, :] >= case["sinks"])
        for h in range(case["kv_heads"]):
            k, v = (_exact_row(s["cache"][where, h, i, off], s["scales"][where, h, i, :, off].t()) for i in (0, 1))
            for g in range(h * group, (h + 1) * group):
                score = s["query"][lo:hi, g].double() @ k.t() * s["scale"]
                out[lo:hi, g] = torch.softmax(score.masked_fill_(hidden, -math.inf), -1) @ v
    return out
