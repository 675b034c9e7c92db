"""The 4-bit cache and its attention where a documented call meets an end: query rows that are not finite and see no key,
starts that fall over a small workspace, numbers next to 2^127,
more rows than one axis of a grid has threads for."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kv4_ref
from qwen35_hip import ops
from test_gpu_kv4 import close, dev, gpu_cache, host, random_cache, same_cache, tables

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


def test_what_a_workspace_held_names_no_place_outside_it():
    """Starts that fall leave rows without an entry of this call, where the workspace may hold anything: a place in the region for
    cut prompts' pieces, which so small a workspace does not have, is not read. What lies behind the workspace, here memory of this
    test's own as large as that region, shows in no row."""
    heads, kvh, dim, page, rows, requests, width = 8, 1, 256, 64, 8, 1000, 20
    table, lens = np.zeros((requests, width), I32), np.full(requests, page * width, I32)
    start = np.array([0, 7] * (requests // 2) + [8], I32)   # the last row is the last request's alone, whose pieces never run
    need = ops.attn_kv4_workspace_bytes(rows, requests, heads, kvh, dim)
    region = 2 * 256 * 128 * dim * 4
    memory = torch.full(((need + region) // 4 + 4096,), 3.0, device="cuda")
    info = memory[(need - 512) // 4:need // 4].view(torch.int32).view(64, 2)   # a place and a number of pieces for each pair
    places = (need - 512) // (dim * 4 + 8) // 8 * 8   # sums of dim floats and 8 bytes of statistics each
    out = torch.full((rows, heads, dim), 7.0, device="cuda")
    q = torch.zeros((rows, heads, dim), device="cuda")
    cache = ops.kv4_cache(2, kvh, dim, page)
    for first in (places - 8, places, places + 5, places + 256 * 128 - 1):
        for pieces in (2, 3, 200):
            info[:, 0], info[:, 1] = first, pieces
            memory[need // 4:] = 3.0
            ops.attn_kv4_rows(q, cache, dev(table), dev(start), dev(lens), out=out, workspace=memory.view(torch.uint8)[:need])
            torch.cuda.synchronize()
            assert not bool((out == 3.0).any()) and not bool((out == 1.0).any()), (first, pieces)


@pytest.mark.parametrize("dim", [64, 256])
def test_values_next_to_two_to_the_127_read_back(dim):
    """15 scale passes the largest fp32 number where a group reaches from -2^127 to 2^127; min + 15 scale does not."""
    ref = kv4_ref.Cache(1, 1, 8, dim)
    cache = gpu_cache(ref)
    most = np.nextafter(F32(2.0 ** 127), F32(0))
    x = np.random.default_rng(dim).uniform(-1, 1, (3, 1, dim)).astype(F32) * most
    x[:, :, ::7], x[:, :, 3::7] = -most, most
    x[1] *= F32(0.99)
    x[2, 0, 0::64] = 0.5 * most
    slots = np.arange(3, dtype=I32)
    ops.kv4_store_rows(dev(x), dev(x), dev(slots), cache)
    ref.store(0, x, slots)
    ref.store(1, x, slots)
    for w, got in enumerate(host(t) for t in ops.kv4_read_rows(cache, dev(slots))):
        assert np.array_equal(got, ref.values(w, slots).astype(F32)) and np.all(np.isfinite(got))


def test_store_of_more_rows_than_one_axis_of_a_grid_takes():
    """2^26 + 20 rows, all but a few without a slot."""
    rows, dim, page = (1 << 26) + 20, 64, 16
    ref = kv4_ref.Cache(4, 1, page, dim)
    cache = gpu_cache(ref)
    at = np.concatenate([[0, 9, 1 << 20, (1 << 25) + 3, (1 << 26) - 9], np.arange((1 << 26) - 4, rows)])
    slots = np.concatenate([[40, 1, 7, 50, 33], 8 + np.arange(24)]).astype(I32)
    small = np.random.default_rng(3).standard_normal((len(at), 1, dim)).astype(F32)
    x = torch.empty((rows, 1, dim), device="cuda")
    x[dev(at)] = dev(small)
    where = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    where[dev(at)] = dev(slots)
    ops.kv4_store_rows(x, x, where, cache)
    ref.store(0, small, slots)
    ref.store(1, small, slots)
    same_cache(cache, ref)
