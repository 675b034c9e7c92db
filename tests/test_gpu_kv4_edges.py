"""The 4-bit cache and its attention where a documented call meets an end: query rows that are not finite and see no key,
starts that fall over a small workspace, numbers next to 2^127, more rows than one axis of a grid has threads for, starts that
leave the step, thousands of requests, tables that could hold a thousand million tokens."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kv4_ref
from qwen35_hip import ops
from test_gpu_kv4 import attention_case, close, dev, gpu_cache, host, random_cache, same_cache, tables

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


@pytest.mark.parametrize("lens,width", [((64, -5, 64, 1000), 4), ((3000, -5, 2500, 1 << 30), 200)])
def test_rows_of_starts_that_leave_the_step(lens, width):
    """Starts before the first row and behind the last, a negative length, and a length past the table row of a request that has
    no rows: the rows of each request, in one launch or by pieces."""
    r = np.random.default_rng(width)
    page, heads, kvh, dim = 16, 4, 2, 64
    true = [lens[0], 0, lens[2], 0]
    table, pages = tables(r, true, page, width)
    ref = random_cache(r, pages, kvh, page, dim)
    q = r.standard_normal((12, heads, dim)).astype(F32)
    start = [-7, 3, 6, 2 ** 31 - 1, 2 ** 31 - 1]
    got = host(ops.attn_kv4_rows(dev(q), gpu_cache(ref), dev(table), dev(start, I32), dev(lens, I32)))
    close(got, *kv4_ref.attention(q, ref, table, [0, 3, 6, 12, 12], true))


def test_rows_of_one_request_where_starts_fall():
    """Requests that share some rows: those that one request alone has are right."""
    r = np.random.default_rng(12)
    page, heads, kvh, dim = 16, 4, 2, 64
    table, pages = tables(r, [64] * 4, page)
    ref = random_cache(r, pages, kvh, page, dim)
    q = r.standard_normal((12, heads, dim)).astype(F32)
    got = host(ops.attn_kv4_rows(dev(q), gpu_cache(ref), dev(table), dev([0, 5, 3, 99, 4], I32), dev([64] * 4, I32)))
    for b, first, rows in ((0, 0, [0, 1, 2]), (2, 3, [5, 6, 7, 8, 9, 10, 11])):
        n = 5 if b == 0 else 9
        close(got[rows], *kv4_ref.attention(q[rows], ref, np.repeat(table[b:b + 1], len(rows), 0), range(len(rows) + 1),
                                            [64 - n + row - first + 1 for row in rows]))


@pytest.mark.parametrize("requests,width", [(1025, 4), (1100, 60), (4096, 4), (4096, 60)])
@pytest.mark.parametrize("page", [16, 64])
def test_more_requests_than_are_held_in_registers(requests, width, page):
    """Most of them idle, some of the live ones past 1024, alone and with a few rows each; short tables and long ones."""
    r = np.random.default_rng(requests + width)
    lens, fresh = np.zeros(requests, int), np.zeros(requests, int)
    live = np.concatenate([[0, 63, 64, requests - 1, 1024], r.choice(np.arange(65, 1023), 20, replace=False)])
    lens[live] = r.integers(1, width * page, len(live))
    fresh[live] = np.minimum(lens[live], r.integers(1, 4, len(live)))
    attention_case(r, lens.tolist(), fresh.tolist(), 8, 2, 64, page, pad=1, width=width)


def close_in_some_rows(r, got, q, ref, table, start, lens, some):
    """`some` random rows of each request (its first and last among them) against the 64-bit form, a row a request."""
    rows, of, seen = [], [], []
    for b, total in enumerate(lens):
        n = start[b + 1] - start[b]
        for i in sorted({0, n - 1, *r.integers(0, n, some).tolist()}) if n else ():
            rows.append(start[b] + i)
            of.append(b)
            seen.append(total - n + i + 1)
    close(got[rows], *kv4_ref.attention(q[rows], ref, table[of], range(len(rows) + 1), seen))


def prompts(r, lens, fresh, heads, kvh, dim, page, width):
    table, pages = tables(r, lens, page, width)
    ref = random_cache(r, pages, kvh, page, dim)
    start = np.concatenate([[0], np.cumsum(fresh)]).astype(int)
    q = r.standard_normal((start[-1], heads, dim)).astype(F32)
    got = host(ops.attn_kv4_rows(dev(q), gpu_cache(ref), dev(table), dev(start, I32), dev(lens, I32)))
    close_in_some_rows(r, got, q, ref, table, start.tolist(), lens, 6)


@pytest.mark.parametrize("at", [1024, 2000, 4095])
def test_a_prompt_past_the_requests_in_registers(at):
    """A chunk too heavy to be a light call, one of few rows and single tokens, among 4096 requests."""
    r = np.random.default_rng(at)
    lens, fresh = np.zeros(4096, int), np.zeros(4096, int)
    lens[[3, 1023, 3000, at]], fresh[[3, 1023, 3000, at]] = (700, 90, 64, 640), (1, 12, 1, 600)
    prompts(r, lens.tolist(), fresh.tolist(), 16, 2, 64, 16, 48)


@pytest.mark.parametrize("width", [65535, 65536, 1 << 18, 1 << 20])
@pytest.mark.parametrize("lens,fresh,heads,kvh,dim", [
    ([5000, 33], [140, 1], 64, 2, 64),                 # few row tiles, in pieces
    ([700, 2100, 90], [600, 300, 1], 16, 2, 64),       # row tiles short and long
    ([4000, 2200], [300, 200], 64, 16, 64),            # hundreds of them, one line
    ([1500], [170], 48, 3, 256),
])
def test_prompts_over_tables_of_up_to_a_thousand_million_tokens(lens, fresh, heads, kvh, dim, width):
    """A line of tiles counts steps of 2, 8 and 32 tiles there, so that its length stays in 32 bits."""
    prompts(np.random.default_rng(width + dim), lens, fresh, heads, kvh, dim, 1024, width)
