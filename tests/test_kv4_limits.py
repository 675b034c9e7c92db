"""Bounds that the documentation of the 4-bit cache gives. Calls of its attention whose launch would have 2^32 threads along one
axis, which runs short without an error, are refused before any launch, on the CPU; pointers here are never followed."""

from __future__ import annotations

import ctypes

import kv4_ref
import numpy as np
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


def test_how_far_a_stored_value_may_be_off():
    """Half a step; a step is a fifteenth of the range from the minimum, which is rounded down by less than 1/128 of its size, and
    is rounded up by at most 1/128. A group far from zero comes near that, and past half a fifteenth of its own range."""
    r = np.random.default_rng(0)
    x = (r.uniform(-1, 1, (3000, 1)) * 10.0 ** r.integers(-3, 4, (3000, 1)) + r.uniform(0, 1, (3000, 64))).astype(np.float32)
    x[0] = r.uniform(100.3, 100.4, 64)
    codes, scale, low = kv4_ref.quantize(x)
    v = x.astype(np.float64)
    off = np.abs(low[:, None] + scale[:, None] * codes - v).max(-1)
    span = v.max(-1) - v.min(-1)
    bound = 0.5 * (span + np.abs(v.min(-1)) / 128) / 15 * (1 + 1 / 128)
    assert np.all(off <= bound * (1 + 2.0 ** -40))
    assert off[0] > span[0] / 30
