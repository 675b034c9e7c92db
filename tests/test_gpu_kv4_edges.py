"""The 4-bit cache and its attention where a documented call meets an end: query rows that are not finite and see no key."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kv4_ref
from qwen35_hip import ops
from test_gpu_kv4 import close, dev, gpu_cache, host, random_cache, tables

pytestmark = pytest.mark.gpu
F32, I32 = np.float32, np.int32


@pytest.mark.parametrize("heads,kvh,dim,n,total,page", [
    (16, 2, 256, 3, 2, 16), (8, 2, 64, 12, 5, 64),     # by blocks of 8 (row, head) pairs
    (64, 2, 64, 140, 101, 16), (64, 2, 128, 140, 101, 64), (96, 3, 256, 140, 103, 8),   # by row tiles of 128 pairs, too many to be light
    (128, 128, 64, 300, 250, 16),                      # the same, cut as one line of tiles
])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_rows_without_keys_are_zeros_whatever_their_query_holds(heads, kvh, dim, n, total, page, value):
    """kv_len below the request's rows: the first n - total rows see nothing. One of them, the last of them and the first row
    that sees a key have an infinity or NaN in the query of one head: zeros where no key is seen, NaN in that one head where
    one is, and what a clean query gives everywhere else."""
    r = np.random.default_rng(heads + n)
    table, pages = tables(r, [total], page)
    ref = random_cache(r, pages, kvh, page, dim)
    clean = r.standard_normal((n, heads, dim)).astype(F32)
    q, bad = clean.copy(), np.zeros((n, heads), bool)
    for row, head in ((0, 0), (n - total - 1, heads - 1), (n - total, heads // 2)):
        q[row, head, 5] = value
        bad[row, head] = row >= n - total
    got = host(ops.attn_kv4_rows(dev(q), gpu_cache(ref), dev(table), dev([0, n], I32), dev([total], I32)))
    assert np.all(got[:n - total] == 0)
    assert np.array_equal(np.isnan(got).all(-1), bad) and np.array_equal(np.isnan(got).any(-1), bad)
    some = sorted({*range(max(n - total - 2, 0), min(n - total + 4, n)), n - 1, *r.integers(0, n, 6).tolist()})
    want, tol = kv4_ref.attention(clean[some], ref, np.repeat(table, len(some), 0), range(len(some) + 1),
                                  [total - n + row + 1 for row in some])
    good = ~bad[some]
    close(got[some][good], want[good], tol[good])
