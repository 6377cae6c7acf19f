"""The definition of the paged 4-bit cache itself (oracle/paged.py), and what the C entry points refuse before they
touch a device."""
import ctypes

import numpy as np
import pytest

from oracle import paged


def test_levels_and_ties():
    x = np.zeros(32)
    x[:14] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.0, -0.25, -5, 0.26, 5.01, 0.74]
    code, byte = paged.encode(x)
    assert byte.tolist() == [127]
    got = paged.decode(code, byte)[:14]
    assert got.tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 0, 0, -4, 0.5, 6, 0.5]
    assert np.signbit(got[8]) and np.signbit(got[9])


@pytest.mark.parametrize("e", [-127, -126, -3, 0, 5, 100, 125])
def test_power_of_two_of_a_block(e):
    x = np.zeros(32)
    x[3] = 7 * 2.0**e * (1 - 2**-23)
    code, byte = paged.encode(x)
    assert byte[0] == e + 127 and paged.decode(code, byte)[3] == 6 * 2.0**e
    x[3] = -7 * 2.0**e
    code, byte = paged.encode(x)
    assert byte[0] == e + 128 and paged.decode(code, byte)[3] == -8 * 2.0**e


def test_broken_and_empty_blocks():
    x = np.zeros((3, 64))
    x[0, 40], x[1, 2] = np.nan, -np.inf
    code, byte = paged.encode(x)
    assert byte.tolist() == [[0, 255], [255, 0], [0, 0]] and not code.any()
    assert np.isnan(paged.decode(code, byte)).sum() == 64


def test_rounding_error_is_half_a_step():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((500, 32)) * np.exp2(rng.integers(-20, 20, size=(500, 1)))
    code, byte = paged.encode(x)
    power = np.exp2(byte.astype(float) - 127)
    y = np.abs(x) / power
    step = np.where(y < 2, 0.5, np.where(y < 4, 1, 2))
    assert (np.abs(paged.decode(code, byte) - x) <= step * power / 2 + 1e-300).all()


def test_plan_of_a_small_batch():
    table = np.full((3, 4), -1, np.int32)
    table[1, 0] = 9
    starts, lens, pos, slots, counts = paged.plan(np.array([0, 5, 0]), np.array([17, 2, 0]), table, np.array([4, 2, 7]),
                                                  16, 21)
    assert starts.tolist() == [0, 17, 19, 19] and lens.tolist() == [17, 7, 0] and counts.tolist() == [19, 2]
    assert table.tolist() == [[4, 2, -1, -1], [9, -1, -1, -1], [-1] * 4]
    assert slots.tolist() == list(range(64, 80)) + [32, 149, 150, -1, -1]
    assert pos.tolist() == list(range(17)) + [5, 6, -1, -1]


def _cache(cabi, **kw):
    c = dict(cache=4096, scales=8192, pages=2, cache_page_stride=2 * 16 * 128 * 8, scales_page_stride=2 * 16 * 8 * 8,
             kv_heads=8, dim=128, page=16)
    c.update(kw)
    return cabi.PagedCache(*[c[f] for f, _ in cabi.PagedCache._fields_])


def _refused(cabi, rc, text, code=-1):
    assert rc == code and text in cabi.load().shmt_last_error().decode()


@pytest.mark.parametrize("bad, text", [
    (dict(dim=96), "64, 128 or 256"), (dict(page=8), "a page must hold"), (dict(page=48), "a page must hold"),
    (dict(kv_heads=0), "number of heads"), (dict(pages=-1), "number of pages"), (dict(cache_page_stride=1024), "overlap"),
    (dict(scales_page_stride=64), "overlap"), (dict(cache=None), "null"), (dict(cache=4104), "on 16 bytes"),
    (dict(scales_page_stride=4104), "on 16 bytes")])
def test_cache_descriptions_that_are_refused(cabi, bad, text):
    lib, c = cabi.load(), _cache(cabi, **bad)
    _refused(cabi, lib.shmt_page_set(ctypes.byref(c), None, 8, 0, None, 0, 0, None, 0, 0, 2, None), text)
    _refused(cabi, lib.shmt_page_fetch(ctypes.byref(c), None, 8, 0, None, None, 2, None), text)
    _refused(cabi, lib.shmt_page_attention(ctypes.byref(c), None, 0, 0, 2, 0, 8, None, 0, 0, None, None, 4, 0, 1.0, 0, 0,
                                           0, None, None, None, 0, None), text)


def test_rows_that_are_refused(cabi):
    lib, c = cabi.load(), _cache(cabi)
    def set_(n=1, width=8, k=4096, stride=1024, kind=2, slots=16):
        return lib.shmt_page_set(ctypes.byref(c), slots, width, n, k, stride, 128, 8192, 1024, 128, kind, None)
    _refused(cabi, set_(n=-1), ">= 0")
    _refused(cabi, set_(width=2), "int32 or int64")
    _refused(cabi, set_(kind=3), "element type")
    _refused(cabi, set_(k=None), "null")
    _refused(cabi, set_(slots=None), "null")
    _refused(cabi, set_(k=4098), "16 bytes")
    _refused(cabi, set_(stride=1028), "16 bytes")
    _refused(cabi, lib.shmt_page_set(None, 16, 8, 1, 4096, 1024, 128, 8192, 1024, 128, 2, None), "cache is null")
    assert set_(n=0) == 0


def test_plans_that_are_refused(cabi):
    lib = cabi.load()
    def plan(cached=16, width=8, n=1, table=4096, w=4, stride=4, n_free=3, page=16, most=4, starts=64, scratch_bytes=1 << 20,
             free=32):
        return lib.shmt_page_plan(cached, 16, width, n, table, w, stride, free, n_free, page, most, starts, 16, 16, 16, 16,
                                  16, scratch_bytes, None)
    for kw, text in ((dict(n=-1), "requests"), (dict(width=3), "int32 or int64"), (dict(page=24), "a page must hold"),
                     (dict(most=1 << 31), "max_tokens"), (dict(stride=3), "narrow"), (dict(table=None), "null"),
                     (dict(cached=None), "null"), (dict(starts=None), "null"), (dict(n_free=-1), ">= 0"),
                     (dict(free=None), "null")):
        _refused(cabi, plan(**kw), text)
    if lib.shmt_page_plan_scratch_bytes(100000) > 0:
        _refused(cabi, plan(n=100000, scratch_bytes=0), "scratch", code=-4)


def test_attention_that_is_refused(cabi):
    lib, c = cabi.load(), _cache(cabi)
    def attend(q=4096, stride=4096, kind=2, tokens=3, heads=32, table=64, width=4, tstride=4, starts=64, lens=64, n=2, lb=4,
               scale=0.1, window=0, sinks=0, most=0, out=4096):
        return lib.shmt_page_attention(ctypes.byref(c), q, stride, 128, kind, tokens, heads, table, width, tstride, starts,
                                       lens, lb, n, scale, window, sinks, most, out, None, None, 0, None)
    for kw, text in ((dict(kind=0), "float16 or bfloat16"), (dict(heads=12), "evenly"), (dict(heads=0), "evenly"),
                     (dict(tokens=-1), "query rows"), (dict(n=-2), "requests"), (dict(lb=1), "int32 or int64"),
                     (dict(window=-1), ">= 0"), (dict(sinks=-1), ">= 0"), (dict(most=-1), ">= 0"),
                     (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(q=None), "null"),
                     (dict(out=None), "null"), (dict(starts=None), "null"), (dict(table=None), "null"),
                     (dict(tstride=2), "narrow"), (dict(q=4100), "16 bytes"), (dict(stride=4100), "16 bytes"),
                     (dict(out=4104), "16 bytes"), (dict(width=1 << 30, tstride=1 << 30), "too many tokens")):
        _refused(cabi, attend(**kw), text)
    assert attend(tokens=0) == 0
