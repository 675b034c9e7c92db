"""Host validation of the rotation by several axes, the 4-bit cache and its attention: refused before any launch, on the
CPU. Pointers here are never followed. And the 64-bit forms of the quantization against its definition."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import kv4_ref
from qwen35_hip import _lib

P, ODD, NUL = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 4), None
FAR = ctypes.c_void_p(1 << 32)
INV, OK = _lib.STATUS_INVALID_ARGUMENT, _lib.STATUS_OK


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(lib, status, words):
    assert status == INV
    assert words in lib.qwen_last_error().decode(), lib.qwen_last_error().decode()


def test_mrope(lib):
    def call(sections=(11, 11, 10), **kw):
        a = dict(q=P, k=FAR, qw=P, kw=P, pos=P, sections=(ctypes.c_int32 * max(len(sections), 1))(*sections),
                 axes=len(sections), interleaved=1, rows=3, qh=16, kh=2, hd=256, theta=1e7, eps=1e-6, stream=NUL)
        a.update(qw=ctypes.c_void_p(1 << 33), kw=ctypes.c_void_p(1 << 34), pos=ctypes.c_void_p(1 << 35))
        a.update(kw)
        return lib.qwen_attn_qk_norm_mrope_rows(*a.values())
    refused(lib, call(()), "axes")
    refused(lib, call((1, 1, 1, 1, 1)), "axes")
    refused(lib, call(sections=(8,), axes=1, rows=-1), "negative")
    refused(lib, call((4, -1, 8)), "negative")
    refused(lib, call((0, 0, 0)), "pairs")
    refused(lib, call((64, 64, 1)), "pairs")
    refused(lib, call((64, 60, 4), hd=254), "pairs")
    refused(lib, call((2 ** 31 - 1, 2 ** 31 - 1, 2)), "pairs")
    refused(lib, call(hd=0), "head_dim")
    for theta in (0.0, -1.0, float("nan"), float("inf")):
        refused(lib, call(theta=theta), "theta")
    refused(lib, call(rows=1 << 28), "2^31")
    for name in ("q", "k", "qw", "kw", "pos"):
        refused(lib, call(**{name: NUL}), "null")
    refused(lib, call(k=P), "overlap")
    refused(lib, call(pos=P), "overlap")
    refused(lib, call(kw=FAR), "overlap")
    assert call(rows=0, q=NUL) == OK and call(qh=0, kh=0, q=NUL) == OK


CACHE = dict(kc=P, vc=P, ks=P, km=P, vs=P, vm=P, pages=8, page=64, heads=2, dim=256)


@pytest.mark.parametrize("bad,words", [
    (dict(kc=NUL), "null cache"), (dict(vs=NUL), "null cache"), (dict(km=NUL), "null cache"), (dict(vm=NUL), "null cache"),
    (dict(vc=ODD), "aligned"), (dict(ks=ODD), "aligned"), (dict(vm=ODD), "aligned"), (dict(pages=0), "pages"),
    (dict(pages=1 << 26), "pages"), (dict(page=24), "power of two"), (dict(page=4), "power of two"),
    (dict(page=2048), "power of two"), (dict(heads=0), "KV heads"), (dict(heads=65536), "KV heads"), (dict(dim=96), "head dim"),
    (dict(dim=0), "head dim"),
])
def test_cache_shapes(lib, bad, words):
    c = {**CACHE, **bad}
    ptrs, (pages, page, heads, dim) = list(c.values())[:6], list(c.values())[6:]
    refused(lib, lib.qwen_kv4_store_rows(P, P, 1 << 25, 1 << 25, P, 3, *ptrs, pages, page, heads, dim, NUL), words)
    refused(lib, lib.qwen_kv4_read_rows(*ptrs, pages, page, heads, dim, P, 3, P, P, NUL), words)
    if heads:
        refused(lib, lib.qwen_attn_kv4_rows(P, *ptrs, pages, page, P, 4, P, P, 2, NUL, P, 3, 16, heads, dim, P, 1 << 40, NUL),
                words)


def test_store_and_read(lib):
    c = tuple(CACHE.values())
    st = lambda k=P, v=P, ks=512, vs=512, slots=P, rows=3: lib.qwen_kv4_store_rows(k, v, ks, vs, slots, rows, *c, NUL)
    refused(lib, st(rows=-1), "negative")
    refused(lib, st(k=NUL), "null")
    refused(lib, st(slots=NUL), "null")
    refused(lib, st(vs=511), "strides")
    refused(lib, st(ks=-512), "strides")
    assert st(k=NUL, v=NUL, slots=NUL, rows=0) == OK
    rd = lambda slots=P, rows=3, k=P, v=FAR: lib.qwen_kv4_read_rows(*c, slots, rows, k, v, NUL)
    refused(lib, rd(rows=-1), "negative")
    refused(lib, rd(rows=1 << 25), "exceed one call")
    refused(lib, rd(k=ODD), "aligned")
    refused(lib, rd(v=NUL), "null")
    refused(lib, rd(v=P), "overlap")
    assert rd(slots=NUL, rows=0, k=NUL, v=NUL) == OK


def test_attention(lib):
    need = lib.qwen_attn_kv4_workspace_bytes

    def call(**kw):
        a = dict(q=P, **{k: CACHE[k] for k in ("kc", "vc", "ks", "km", "vs", "vm")}, pages=8, page=64, table=P, max_pages=4,
                 start=P, len=P, requests=2, gate=NUL, out=ctypes.c_void_p(1 << 21), rows=3, heads=16, kv=2, dim=256, ws=P,
                 bytes=1 << 40, stream=NUL)
        a.update(kw)
        return lib.qwen_attn_kv4_rows(*a.values())
    refused(lib, call(heads=15), "query heads")
    refused(lib, call(heads=0), "query heads")
    refused(lib, call(rows=-1), "negative")
    refused(lib, call(requests=4097), "at most 4096")
    refused(lib, call(max_pages=1 << 30), "table rows")
    refused(lib, call(max_pages=(1 << 24) + 1), "table rows")
    refused(lib, call(rows=1 << 21), "exceed one call")
    refused(lib, call(out=P), "out is q")
    refused(lib, call(gate=ctypes.c_void_p((1 << 21) + 16)), "out of place")
    for name in ("q", "out", "gate"):
        refused(lib, call(**{name: ODD}), "aligned")
    for name in ("q", "out", "start", "len", "table"):
        refused(lib, call(**{name: NUL}), "null")
    refused(lib, call(ws=NUL), "workspace")
    refused(lib, call(ws=ODD), "workspace")
    refused(lib, call(bytes=need(3, 2, 16, 2, 256) - 1), "workspace")
    assert call(rows=0, q=NUL) == OK and call(requests=0, start=NUL) == OK
    assert need(0, 2, 16, 2, 256) == 0 and need(3, 0, 16, 2, 256) == 0 and need(3, 2, 15, 2, 256) == 0
    assert need(3, 2, 16, 2, 256) > 0


def test_workspace_grows_with_rows_and_requests(lib):
    """One for some rows and requests serves fewer of either."""
    need = lib.qwen_attn_kv4_workspace_bytes
    for heads, kv, dim in ((16, 2, 256), (24, 8, 128), (12, 12, 64), (7, 1, 256)):
        rows = [1, 2, 3, 4, 5, 8, 16, 32, 33, 63, 64, 65, 128, 129, 500, 1024, 1025, 5000]
        for requests in (1, 2, 64, 65, 4096):
            sizes = [need(n, requests, heads, kv, dim) for n in rows]
            assert sizes == sorted(sizes)
        for n in rows:
            sizes = [need(n, requests, heads, kv, dim) for requests in (1, 2, 5, 33, 64, 65, 1000, 4096)]
            assert sizes == sorted(sizes)


def test_quantization_of_the_reference():
    """kv4_ref.quantize against its definition: the neighbours of scale and min, and values within half a step."""
    r = np.random.default_rng(0)
    x = (r.standard_normal((400, 64)) * 10.0 ** r.integers(-20, 20, (400, 1)) + r.standard_normal((400, 1))).astype(np.float32)
    codes, scale, low = kv4_ref.quantize(x)
    up = lambda v: (np.asarray(v, np.float32).view(np.int32) + 0x10000).view(np.float32).astype(np.float64)   # away from zero
    down = lambda v: (np.asarray(v, np.float32).view(np.int32) - 0x10000).view(np.float32).astype(np.float64)
    small, large = x.min(-1).astype(np.float64), x.max(-1).astype(np.float64)
    assert np.all(low <= small) and np.all(np.where(low < 0, down(low), up(low)) > small)
    assert np.all(scale >= (large - low) / 15) and np.all(down(scale) < (large - low) / 15)
    assert codes.min() == 0 and codes.max() == 15
    assert np.all(np.abs(low[:, None] + scale[:, None] * codes - x) <= 0.5 * scale[:, None] * (1 + 2.0 ** -40))
