"""Calls of the 4-bit attention whose launch would have 2^32 threads along one axis, which runs short without an error: refused
before any launch, on the CPU. Pointers here are never followed."""

from __future__ import annotations

import ctypes

import pytest

from qwen35_hip import _lib

P, OUT, BIG = ctypes.c_void_p(1 << 20), ctypes.c_void_p(1 << 40), 1 << 50


@pytest.mark.parametrize("rows,requests,heads,kvh,max_pages", [
    (129, 129, 65535, 65535, 4), (256, 256, 65535, 65535, 4),        # short tables: eight waves a row and KV head
    (256, 256, 65535, 65535, 64), (4096, 4096, 4096, 4096, 64),      # long ones: four
])
def test_single_rows_of_too_many_heads(rows, requests, heads, kvh, max_pages):
    lib = _lib.load()
    status = lib.qwen_attn_kv4_rows(P, *[P] * 6, 8, 64, P, max_pages, P, P, requests, None, OUT, rows, heads, kvh, 64, P, BIG, None)
    assert status == _lib.STATUS_INVALID_ARGUMENT
    assert "exceed one call" in lib.qwen_last_error().decode()
