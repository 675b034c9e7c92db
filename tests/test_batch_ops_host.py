"""Host validation of the operators of several requests and of many tokens' experts: refused before any launch, on the
CPU. Pointers here are never followed."""

from __future__ import annotations

import ctypes

import pytest

from qwen35_hip import _lib

P, ODD, NUL = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 4), None
INV, OK, UNS = _lib.STATUS_INVALID_ARGUMENT, _lib.STATUS_OK, _lib.STATUS_UNSUPPORTED_TYPE


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(lib, status, words):
    assert status == INV
    assert words in lib.qwen_last_error().decode(), lib.qwen_last_error().decode()


def test_plan(lib):
    def call(**kw):
        a = dict(cached=P, fresh=P, requests=4, table=P, max_pages=8, free=P, n_free=9, head=P, head_out=P, page=64, rows=5,
                 start=P, len=P, slots=P, pos=P, stream=NUL)
        a.update(kw)
        return lib.qwen_kv8_plan(*a.values())
    refused(lib, call(requests=-1), "requests")
    refused(lib, call(requests=4097), "at most 4096")
    for page in (0, 4, 48, 2048, -8):
        refused(lib, call(page=page), "power of two")
    refused(lib, call(rows=-1), "negative")
    refused(lib, call(max_pages=1 << 30), "table rows")
    for name in ("cached", "fresh", "table", "head", "head_out", "start", "len"):
        refused(lib, call(**{name: NUL}), "null")
    refused(lib, call(free=NUL), "free list")
    refused(lib, call(slots=NUL), "null slots")


CACHE = dict(kc=P, vc=P, ks=P, vs=P, pages=8, page=64, heads=2, dim=256)


@pytest.mark.parametrize("bad,words", [
    (dict(kc=NUL), "null cache"), (dict(vs=NUL), "null cache"), (dict(vc=ODD), "aligned"), (dict(pages=0), "pages"),
    (dict(pages=1 << 26), "pages"), (dict(page=24), "power of two"), (dict(heads=0), "KV heads"), (dict(dim=96), "head dim"),
])
def test_cache_shapes(lib, bad, words):
    c = {**CACHE, **bad}
    kc, vc, ks, vs, pages, page, heads, dim = c.values()
    refused(lib, lib.qwen_kv8_store_rows(P, P, 512, 512, P, 3, kc, vc, ks, vs, pages, page, heads, dim, NUL), words)
    refused(lib, lib.qwen_kv8_read_rows(kc, vc, ks, vs, pages, page, heads, dim, P, 3, P, P, NUL), words)
    if heads:
        refused(lib, lib.qwen_attn_kv8_rows(P, kc, vc, ks, vs, pages, page, P, 4, P, P, 2, NUL, P, 3, 16, heads, dim, P, 1 << 40,
                                            NUL), words)


def test_store_and_read(lib):
    c = tuple(CACHE.values())
    st = lambda k=P, v=P, ks=512, vs=512, slots=P, rows=3: lib.qwen_kv8_store_rows(k, v, ks, vs, slots, rows, *c, NUL)
    refused(lib, st(rows=-1), "negative")
    refused(lib, st(k=NUL), "null")
    refused(lib, st(slots=NUL), "null")
    refused(lib, st(vs=511), "strides")
    assert st(k=NUL, v=NUL, slots=NUL, rows=0) == OK
    rd = lambda slots=P, rows=3, k=P, v=P: lib.qwen_kv8_read_rows(*c, slots, rows, k, v, NUL)
    refused(lib, rd(rows=-1), "negative")
    refused(lib, rd(k=ODD), "aligned")
    refused(lib, rd(v=NUL), "null")
    assert rd(slots=NUL, rows=0, k=NUL, v=NUL) == OK


def test_attention(lib):
    need = lib.qwen_attn_kv8_workspace_bytes

    def call(**kw):
        a = dict(q=P, kc=P, vc=P, ks=P, vs=P, pages=8, page=64, table=P, max_pages=4, start=P, len=P, requests=2, gate=NUL,
                 out=ctypes.c_void_p(1 << 21), rows=3, heads=16, kv=2, dim=256, ws=P, bytes=1 << 40, stream=NUL)
        a.update(kw)
        return lib.qwen_attn_kv8_rows(*a.values())
    refused(lib, call(heads=15), "query heads")
    refused(lib, call(heads=0), "query heads")
    refused(lib, call(rows=-1), "negative")
    refused(lib, call(requests=4097), "at most 4096")
    refused(lib, call(max_pages=1 << 30), "table rows")
    refused(lib, call(max_pages=(1 << 24) + 1), "table rows")
    refused(lib, call(rows=1 << 21), "exceed one call")
    refused(lib, call(out=P), "out is q")
    for name in ("q", "out", "gate"):
        refused(lib, call(**{name: ODD}), "aligned")
    for name in ("q", "out", "start", "len", "table"):
        refused(lib, call(**{name: NUL}), "null")
    refused(lib, call(ws=NUL), "workspace")
    refused(lib, call(ws=ODD), "workspace")
    refused(lib, call(bytes=need(3, 2, 16, 2, 256) - 1), "workspace")
    assert call(rows=0, q=NUL) == OK and call(requests=0, start=NUL) == OK
    assert need(0, 2, 16, 2, 256) == 0 and need(3, 0, 16, 2, 256) == 0 and need(3, 2, 15, 2, 256) == 0
    assert need(64, 64, 16, 2, 256) > need(3, 2, 16, 2, 256) > 0


def test_experts(lib):
    need = lib.qwen_moe_experts_rows_workspace_bytes

    def call(**kw):
        a = dict(g=P, u=P, type=12, d=P, down=14, experts=16, order=P, starts=P, w=P, top=8, x=P, rows=3, width=512, inter=256,
                 out=ctypes.c_void_p(1 << 21), ws=P, bytes=1 << 40, stream=NUL)
        a.update(kw)
        return lib.qwen_moe_experts_rows(*a.values())
    refused(lib, call(g=NUL), "not loaded")
    assert call(type=8) == UNS and call(down=0) == UNS
    refused(lib, call(width=500), "multiples of 256")
    refused(lib, call(inter=0), "multiples of 256")
    refused(lib, call(width=(1 << 20) + 256), "exceed 2^20")
    refused(lib, call(experts=1025), "experts")
    refused(lib, call(experts=0), "experts")
    refused(lib, call(rows=-1), "rows")
    refused(lib, call(top=0), "picks")
    refused(lib, call(rows=1 << 22), "picks")
    refused(lib, call(rows=1 << 21, inter=1024), "exceed one call")
    for name in ("order", "starts", "w", "x", "out"):
        refused(lib, call(**{name: NUL}), "null")
    for name in ("g", "u", "d", "x", "out"):
        refused(lib, call(**{name: ODD}), "aligned")
    refused(lib, call(out=P), "out is x")
    refused(lib, call(bytes=need(3, 8, 16, 512, 256) - 1), "workspace")
    refused(lib, call(ws=NUL), "workspace")
    assert call(rows=0, x=NUL) == OK
    assert need(0, 8, 16, 512, 256) == 0 and need(3, 8, 16, 500, 256) == 0 and need(3, 8, 16, 512, 256) > 0
    grp = lambda idx=P, pairs=4, n=16, order=P, starts=P: lib.qwen_moe_group_rows(idx, pairs, n, order, starts, NUL)
    refused(lib, grp(pairs=-1), "pairs")
    refused(lib, grp(pairs=(1 << 24) + 1), "pairs")
    refused(lib, grp(n=0), "experts")
    refused(lib, grp(idx=NUL), "null")
    refused(lib, grp(starts=NUL), "null")
