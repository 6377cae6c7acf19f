"""What the C entry points of trees, kept paths, 8-bit rows and attention over them refuse: arguments are checked before anything
is queued, so this needs no GPU. Addresses are made up and never read."""
import ctypes

import pytest

A = 4096                                                               # an address on 16 bytes


def _view(cabi, **kw):
    v = dict(cache=A, scales=A, pages=10, cache_page_stride=1 << 20, scales_page_stride=1 << 16, kv_heads=2, dim=64, page=16)
    v.update(kw)
    return cabi.PagedCache(*[v[k] for k, _ in cabi.PagedCache._fields_])


def _refused(cabi, rc, text, code=-1):
    assert rc == code and text in cabi.load().shmt_last_error().decode(), cabi.load().shmt_last_error()


def test_page_tree(cabi):
    def call(text, **kw):
        a = dict(parents=A, starts=A, lens=A, len_bytes=4, requests=2, tokens=5, nodes=A, positions=A)
        a.update(kw)
        rc = cabi.load().shmt_page_tree(*a.values(), None)
        _refused(cabi, rc, text)
    call("in [0, 2^30)", tokens=-1)
    call("in [0, 2^30)", tokens=1 << 30)
    call("in [0, 2^31)", requests=-1)
    call("int32 or int64", len_bytes=2)
    call("null", parents=None)
    call("null", nodes=None)
    call("null", lens=None)
    call("16 bytes", nodes=A + 4)
    assert cabi.load().shmt_page_tree(None, None, None, 4, 3, 0, None, None, None) == 0     # no nodes: nothing to do


def test_page_keep(cabi):
    def call(text, view={}, **kw):
        a = dict(cache=ctypes.byref(_view(cabi, **view)), bits=4, layers=2, cl=16 << 20, sl=1 << 20, table=A, width=3, stride=3,
                 starts=A, lens=A, len_bytes=4, requests=2, rows=5, parents=A, tokens=A, picked=A, token_bytes=8, given=None,
                 counts=A, path=A, after=A)
        a.update(kw)
        _refused(cabi, cabi.load().shmt_page_keep(*a.values(), None), text)
    call("null", cache=None)
    call("4 or 8 bits", bits=5)
    call("64, 128 or 256", view=dict(dim=96))
    call("16, 32, 64, 128 or 256 tokens", view=dict(page=48))
    call("pages overlap", bits=8, view=dict(cache_page_stride=2 * 2 * 16 * 32))
    call("layers and heads", layers=-1)
    call("layers and heads", layers=1 << 28)
    call("layer has to begin", cl=(16 << 20) + 8)
    call("layers overlap", cl=16)
    call("layers overlap", sl=0)
    call("in [0, 2^30)", rows=-2)
    call("in [0, 2^31)", requests=1 << 31)
    call("too many requests", requests=1 << 26)
    call("too many tokens", width=1 << 30)
    call("query_starts and kv_lens can", len_bytes=3)
    call("tokens and picked can", token_bytes=1)
    call("counts or next", counts=None)
    call("block_table is null or narrow", table=None)
    call("block_table is null or narrow", stride=2)
    call("parents, tokens", path=None)
    assert cabi.load().shmt_page_keep(ctypes.byref(_view(cabi)), 8, 1, 0, 0, None, 0, 0, None, None, 4, 0, 0, None, None, None, 8,
                                      None, None, None, None, None) == 0


def test_rows_in_8_bits(cabi):
    lib = cabi.load()
    rows = lambda f, bits, view={}, n=3, type=2, keys=A: f(ctypes.byref(_view(cabi, **view)), bits, A, 8, n, keys, *(
        (128, 64, A, 128, 64) if f is lib.shmt_page_set_as else (A,)), type, None)
    for f in (lib.shmt_page_set_as, lib.shmt_page_fetch_as):
        _refused(cabi, rows(f, 16), "4 or 8 bits")
        _refused(cabi, rows(f, 8, dict(cache_page_stride=2 * 2 * 16 * 32)), "pages overlap")
        _refused(cabi, rows(f, 8, type=7), "unknown element type")
        _refused(cabi, rows(f, 8, n=-1), ">= 0")
        _refused(cabi, rows(f, 8, keys=A + 2), "16 bytes")
        _refused(cabi, rows(f, 8, keys=None), "null")
        assert rows(f, 8, n=0) == 0


def test_attention(cabi):
    lib = cabi.load()
    size = lambda bits=8, seen=1, dim=64: lib.shmt_page_attention_as_scratch_bytes(5, 4, 2, bits, seen, dim, 2, 2, 3)
    assert size() > 0 and size(bits=4, seen=0) == lib.shmt_page_attention_scratch_bytes(5, 4, 2, 64, 2, 2, 3)
    for bad in (size(bits=3), size(seen=3), size(seen=-1), size(dim=32)):
        assert bad == -1

    def call(text, view={}, code=-1, **kw):
        a = dict(cache=ctypes.byref(_view(cabi, **view)), bits=8, seen=1, nodes=A, query=A, qt=256, qh=64, type=2, tokens=5, heads=4,
                 table=A, width=3, stride=3, starts=A, lens=A, len_bytes=4, requests=2, scale=0.1, window=0, sinks=0, longest=3,
                 out=A, lse=None, scratch=A, scratch_bytes=1 << 40)
        a.update(kw)
        _refused(cabi, lib.shmt_page_attention_as(*a.values(), None), text, code)
    call("4 or 8 bits", bits=2)
    call("unknown rule", seen=3)
    call("have no window", seen=2, window=5)
    call("nodes is null", nodes=None)
    call("nodes is null or does not begin", nodes=A + 8)
    call("float16 or bfloat16", type=0)
    call("evenly", heads=3)
    call("finite", scale=float("nan"))
    call("pages overlap", view=dict(cache_page_stride=2 * 2 * 16 * 32))
    call("scratch too small", scratch_bytes=10, code=-4)


def test_operators_refuse_tensors_that_are_not_on_the_gpu(capi):
    import torch
    ints = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        capi.page_tree(ints, ints, ints[:2])
    cache = torch.zeros((1, 2, 1, 2, 16, 64), dtype=torch.uint8).view(torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="CUDA"):
        capi.page_keep(cache, torch.zeros((1, 2, 1, 2, 2, 16), dtype=torch.uint8), ints[None], ints, ints[:2], ints, ints, ints)


def test_requests_of_a_step_over_trees(cabi):
    """page_keep has a workgroup for each request, so 2^24 of them are too many; the header says so."""
    view = _view(cabi)
    rc = cabi.load().shmt_page_keep(ctypes.byref(view), 4, 1, 0, 0, A, 3, 3, A, A, 4, 1 << 24, 5, A, A, A, 8, None, A, A, A, None)
    _refused(cabi, rc, "2^24 or more")
