"""The paged 8-bit cache: page bookkeeping, storing and reading rows, attention of several requests' rows.

Integers, codes and scales are compared exactly (they do not depend on how a quotient is evaluated), attention with the
tolerance that tests/kv8_ref.py derives from its roundings."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kv8_ref
from qwen35_hip import _lib, ops

pytestmark = pytest.mark.gpu
F32, I32 = np.float32, np.int32


def dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).cuda()


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


def gpu_cache(ref):
    pages, heads, page, dim = ref.codes[0].shape
    v = ref.codes[1].reshape(pages, heads, page // 8, 8, dim).swapaxes(3, 4)
    return ops.Kv8Cache(dev(ref.codes[0], np.int8), dev(v, np.int8), dev(ref.scales[0], F32), dev(ref.scales[1], F32))


def random_cache(r, pages, heads, page, dim):
    ref = kv8_ref.Cache(pages, heads, page, dim)
    for w in (0, 1):
        ref.codes[w] = r.integers(-127, 128, ref.codes[w].shape).astype(np.float64)
        ref.scales[w] = np.float64(F32(0.02 * 2.0 ** r.uniform(-3, 1, ref.scales[w].shape)))
    return ref


def tables(r, lens, page, width=None):
    """Shuffled pages for lens[b] tokens each: table [requests, width], number of pages (two more than used)."""
    need = [-(-n // page) for n in lens]
    ids = r.permutation(sum(need) + 2)
    table = np.full((len(lens), width or max(max(need, default=1), 1)), -5, I32)   # unused entries are never followed
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, sum(need) + 2


# ------------------------------------------------------------------ page bookkeeping
def run_plan(cached, fresh, table, free, head, page, rows, alias=False):
    t, h = dev(table, I32), dev([head], I32)
    out = h if alias else None
    got = ops.kv8_plan(dev(cached, I32), dev(fresh, I32), t, dev(free, I32), h, page, rows, free_head_out=out)
    start, lens, slots, pos, used = (host(x) for x in got)
    want = kv8_ref.plan(cached, fresh, table, list(free), head, page, rows)
    assert np.array_equal(host(t), want[0])
    for a, b in zip((start, lens, slots, pos), want[1:5]):
        assert a.tolist() == list(b)
    assert used.tolist() == [want[5]]


@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("requests,page", [(0, 16), (1, 8), (3, 16), (64, 64), (65, 32), (1023, 16), (1025, 128), (4096, 8)])
def test_plan(requests, page, alias):
    r = np.random.default_rng(requests + page)
    cached, fresh = r.integers(0, 5 * page, requests), r.integers(0, 4, requests)
    if requests > 2:
        fresh[requests // 2], cached[0], fresh[0] = 3 * page + 1, 0, page
    table = r.integers(0, 1000, (requests, 9)).astype(I32)
    free = r.permutation(3 * requests + 20) + 2000
    run_plan(cached, fresh, table, free, 3, page, int(fresh.sum()) + 5, alias)


@pytest.mark.parametrize("n_free,head", [(0, 0), (4, 0), (7, 3), (12, 12), (12, 50), (12, -3)])
def test_plan_short_of_pages(n_free, head):
    """A request that the free pages do not reach for, and those after it that need one, get none; others still run."""
    cached, fresh = [16, 3, 0, 20, 16, 5, 0], [1, 2, 40, 3, 1, 0, 1]
    table = np.arange(7 * 4, dtype=I32).reshape(7, 4) + 100
    run_plan(cached, fresh, table, np.arange(n_free) + 500, head, 16, 60)


def test_plan_odd_inputs():
    """Negative counts, requests past their table row or past the rows of the step."""
    table = np.arange(6 * 2, dtype=I32).reshape(6, 2)
    run_plan([-4, 30, 31, 33, 0, 2 ** 31 - 100], [1, 2, 5, 0, 33, 2 ** 31 - 1], table, np.arange(30), 0, 16, 50)
    run_plan([0, 0, 0], [10, 10, 10], table[:3], np.arange(30), 0, 16, 25)
    run_plan([5], [0], table[:1], np.arange(3), 1, 16, 0)
    run_plan([0, 0], [3, 1], np.zeros((2, 0), I32), np.arange(3), 1, 16, 4)


# ------------------------------------------------------------------ store, read
def check_codes(cache, ref, slots):
    slots = np.asarray(slots)
    p, o = slots // ref.page, slots % ref.page
    k = host(cache.k).astype(np.float64)
    v = host(cache.v).astype(np.float64).swapaxes(3, 4)
    v = v.reshape(k.shape)
    assert np.array_equal(k[p, :, o], ref.codes[0][p, :, o])
    assert np.array_equal(v[p, :, o], ref.codes[1][p, :, o])
    for got, want in ((cache.k_scale, ref.scales[0]), (cache.v_scale, ref.scales[1])):
        assert np.array_equal(host(got).astype(np.float64)[p], want[p], equal_nan=True)


def grow(r, n, heads, dim):
    """Rows whose sizes vary by powers of ten, so that pages' scales grow while they fill."""
    return (r.standard_normal((n, heads, dim)) * 10.0 ** r.integers(-3, 3, (n, heads, 1))).astype(F32)


@pytest.mark.parametrize("page,heads,dim", [(8, 1, 64), (16, 2, 256), (64, 2, 256), (32, 5, 128), (1024, 3, 64)])
def test_store_in_steps(page, heads, dim):
    """Requests filled by steps of 1 to 2 pages + 3 tokens: scales that grow, codes that are rounded again."""
    r = np.random.default_rng(page + dim)
    steps = [[1, 3, 0, 2 * page + 3], [1, page - 1, 5, 1], [1, 1, 1, 1], [page, 2, 7, 1], [1, 1, page + 1, 9]]
    lens = np.sum(steps, axis=0)
    table, pages = tables(r, lens, page)
    ref = random_cache(r, pages, heads, page, dim)   # pages in use again: old codes and scales must not show
    for w in (0, 1):
        ref.scales[w][:] = 1e30
    cache = gpu_cache(ref)
    at = np.zeros(4, int)
    for fresh in steps:
        slots = np.concatenate([[-1]] + [table[b][t // page] * page + t % page for b in range(4)
                                         for t in [np.arange(at[b], at[b] + fresh[b])]] + [[-7]]).astype(I32)
        k, v = grow(r, len(slots), heads, dim), grow(r, len(slots), heads, dim)
        ops.kv8_store_rows(dev(k), dev(v), dev(slots), cache)
        ref.store(0, k, slots)
        ref.store(1, v, slots)
        at += fresh
        live = np.concatenate([table[b][t // page] * page + t % page for b in range(4) for t in [np.arange(at[b])]])
        check_codes(cache, ref, live)
    read = np.concatenate([live, [-1]]).astype(I32)
    gk, gv = (host(t) for t in ops.kv8_read_rows(cache, dev(read)))
    for w, got in ((0, gk), (1, gv)):
        assert np.array_equal(got[:-1], ref.values(w, live).astype(F32))
        assert np.all(got[-1] == 0)


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 1024, 1025, 2500])
def test_store_long_runs_and_odd_rows(rows):
    """Runs over many pages from the middle of one, past 64 rows of a page, over the switch of the rows per workgroup."""
    r = np.random.default_rng(rows)
    page, heads, dim = 128, 2, 64
    table, pages = tables(r, [rows + 37], page)
    ref = random_cache(r, pages, heads, page, dim)
    cache = gpu_cache(ref)
    t = np.arange(37, 37 + rows)
    slots = (table[0][t // page] * page + t % page).astype(I32)
    k, v = grow(r, rows, heads, dim), grow(r, rows, heads, dim)
    ops.kv8_store_rows(dev(k), dev(v), dev(slots), cache)
    ref.store(0, k, slots)
    ref.store(1, v, slots)
    check_codes(cache, ref, slots)


def test_store_ties_and_borders():
    """Quotients on and next to half steps: the nearest code, ties to even; and codes re-rounded on a tie."""
    page, dim = 8, 64
    ref = kv8_ref.Cache(2, 1, page, dim)
    cache = gpu_cache(ref)
    s = F32(1.0 / 127.0)
    x = np.zeros((page, 1, dim), F32)
    half = (np.arange(62) - 31 + 0.5)
    x[0, 0, 0] = 1.0
    x[0, 0, 2:] = half * s
    x[1, 0, 2:] = np.nextafter((half * s).astype(F32), F32(9))
    x[2, 0, 2:] = np.nextafter((half * s).astype(F32), F32(-9))
    x[3, 0, 2:] = half.astype(F32) / F32(127)
    slots = np.arange(page, dtype=I32)
    ops.kv8_store_rows(dev(x[:5]), dev(x[:5]), dev(slots[:5]), cache)
    for w in (0, 1):
        ref.store(w, x[:5], slots[:5])
    check_codes(cache, ref, slots[:5])
    for scale in (2.0, 2.0, 4.0):   # every odd code is a tie of the halving
        y = np.full((1, 1, dim), scale, F32)
        ops.kv8_store_rows(dev(y), dev(y), dev(slots[5:6]), cache)
        for w in (0, 1):
            ref.store(w, y, slots[5:6])
        check_codes(cache, ref, slots[:6])


@pytest.mark.parametrize("size", [0.0, 1e-45, 1e-38, 1e-30, 3e38])
def test_store_extreme_sizes(size):
    ref = kv8_ref.Cache(1, 2, 16, 64)
    cache = gpu_cache(ref)
    r = np.random.default_rng(1)
    x = (r.uniform(-1, 1, (5, 2, 64)) * size).astype(F32)
    ops.kv8_store_rows(dev(x), dev(-x), dev(np.arange(5), I32), cache)
    ref.store(0, x, np.arange(5))
    ref.store(1, -x, np.arange(5))
    check_codes(cache, ref, np.arange(5))


def test_store_non_finite():
    """An infinity or NaN marks its page and head (keys or values alone) until the page is begun again."""
    ref = kv8_ref.Cache(2, 2, 8, 64)
    cache = gpu_cache(ref)
    x = np.ones((4, 2, 64), F32)
    y = x.copy()
    y[1, 1, 5] = np.inf
    z = x.copy()
    z[2, 0, 9] = np.nan
    for first, k, v in ((0, x, x), (4, y, z), (8, x, y), (0, x, x)):
        slots = np.arange(first, first + 4, dtype=I32)
        ops.kv8_store_rows(dev(k), dev(v), dev(slots), cache)
        ref.store(0, k, slots)
        ref.store(1, v, slots)
        check_codes(cache, ref, slots)
        got = host(ops.kv8_read_rows(cache, dev(slots))[0])
        assert np.array_equal(np.isnan(got), np.isnan(ref.values(0, slots)))


def test_store_strided_unaligned_and_out_of_cache():
    r = np.random.default_rng(5)
    page, heads, dim, rows = 16, 2, 64, 21
    ref = random_cache(r, 3, heads, page, dim)
    cache = gpu_cache(ref)
    wide = r.standard_normal((rows, 3 * heads * dim + 3)).astype(F32)
    w = dev(wide)
    for off in (0, 1):   # 16-byte aligned rows are not the only ones
        kt = w[:, off:off + heads * dim].view(rows, heads, dim)
        vt = w[:, off + 2 * heads * dim:off + 3 * heads * dim].view(rows, heads, dim)
        slots = np.concatenate([np.arange(5, 5 + rows - 3), [48, 2 ** 31 - 1, -1]]).astype(I32)
        ops.kv8_store_rows(kt, vt, dev(slots), cache)
        ref.store(0, host(kt), slots)
        ref.store(1, host(vt), slots)
        check_codes(cache, ref, slots[:rows - 3])
        got = host(ops.kv8_read_rows(cache, dev(slots))[1])
        assert np.all(np.isnan(got[rows - 3:rows - 1])) and np.all(got[rows - 1] == 0)


# ------------------------------------------------------------------ attention
def attention_case(r, lens, fresh, heads, kvh, dim, page, gated=True, pad=0, sigma=1.0, width=None):
    ref_lens = list(lens)
    table, pages = tables(r, ref_lens, page, width)
    ref = random_cache(r, pages, kvh, page, dim)
    rows = int(np.sum(fresh))
    start = np.concatenate([[0], np.cumsum(fresh)]).astype(I32)
    q = (sigma * r.standard_normal((rows + pad, heads, dim))).astype(F32)
    gate = r.standard_normal((rows + pad, heads, dim)).astype(F32) if gated else None
    out = torch.full((rows + pad, heads, dim), 7.0, device="cuda")
    got = host(ops.attn_kv8_rows(dev(q), gpu_cache(ref), dev(table), dev(start), dev(ref_lens, I32),
                                 gate=None if gate is None else dev(gate), out=out))
    want, tol = kv8_ref.attention(q, ref, table, start, ref_lens, gate)
    err = np.abs(got - want)
    assert np.all(err <= tol), (float((err / np.maximum(tol, 1e-300)).max()), np.argwhere(err > tol)[0])
    return got


@pytest.mark.parametrize("heads,kvh,dim", [(16, 2, 256), (1, 1, 64), (12, 4, 128), (40, 2, 64), (7, 1, 256), (24, 8, 128)])
@pytest.mark.parametrize("page", [8, 64])
def test_attention_single_tokens(heads, kvh, dim, page):
    """A row of each request: lengths of one, around the tile of 32 tokens and the page, idle requests between."""
    r = np.random.default_rng(heads + dim)
    lens = [1, 2, 8, 31, 32, 33, 0, 64, 65, 129, 257, 300]
    attention_case(r, lens, [1] * 6 + [0] + [1] * 5, heads, kvh, dim, page, pad=3)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 16, 17, 33, 70])
@pytest.mark.parametrize("heads,kvh,dim,page", [(16, 2, 256, 64), (6, 2, 64, 8), (8, 8, 128, 16)])
def test_attention_rows_of_one_request(n, heads, kvh, dim, page):
    """From the few-row kernel to the many-row one, behind a cached prefix and without one."""
    r = np.random.default_rng(n + dim)
    attention_case(r, [n], [n], heads, kvh, dim, page)
    attention_case(r, [n + 41], [n], heads, kvh, dim, page, gated=False)


def test_attention_prompts_and_tokens_mixed():
    r = np.random.default_rng(3)
    attention_case(r, [300, 70, 40, 129, 5, 200], [1, 70, 0, 50, 5, 2], 16, 2, 256, 32, pad=2)
    attention_case(r, [150, 33, 64], [100, 33, 1], 10, 2, 64, 16)


def test_attention_long_context_in_pieces():
    """Many pieces of one request's keys, joined; and a batch whose pieces differ in number."""
    r = np.random.default_rng(4)
    attention_case(r, [5000], [1], 16, 2, 128, 64)
    attention_case(r, [3000, 1, 700, 2049], [1, 1, 2, 1], 8, 1, 64, 16)


@pytest.mark.parametrize("heads,kvh,dim,page", [(16, 2, 256, 64), (6, 2, 64, 8), (8, 8, 128, 16)])
def test_attention_prompts_in_pieces(heads, kvh, dim, page):
    """Chunks of prompts behind long prefixes: too few row tiles for the card, so that their keys are cut and joined.
    Lengths around the pieces' and tiles' ends; two chunks whose pieces differ in number; single tokens beside them."""
    r = np.random.default_rng(dim)
    for n, before in ((40, 473), (33, 991), (70, 1500), (36, 220)):
        attention_case(r, [before + n], [n], heads, kvh, dim, page, gated=n != 33)
    attention_case(r, [1100, 900, 530, 64], [50, 1, 35, 40], heads, kvh, dim, page, pad=2)


def test_attention_no_more_rows_than_requests():
    """A batch padded to many requests, one of which has most of the rows (the few-row kernel takes them all)."""
    r = np.random.default_rng(33)
    attention_case(r, [700, 0, 90, 1] + [0] * 60, [58, 0, 5, 1] + [0] * 60, 16, 2, 128, 16)
    attention_case(r, [0] * 79 + [130], [0] * 79 + [80], 8, 2, 64, 8, pad=0)


def test_a_cache_stays_over_its_tensors():
    cache = ops.kv8_cache(2, 1, 64, 8)
    with pytest.raises(AttributeError, match="stays over"):
        cache.k = cache.k.clone()


def test_attention_prompts_in_pieces_bad_page():
    """A page outside the cache makes every row of its request NaN that sees it, whichever piece holds it."""
    r = np.random.default_rng(31)
    lens, fresh = [900, 700], [60, 50]
    table, pages = tables(r, lens, 32)
    table[0, 3] = pages + 5
    ref = random_cache(r, pages, 2, 32, 128)
    q = r.standard_normal((110, 16, 128)).astype(F32)
    got = host(ops.attn_kv8_rows(dev(q), gpu_cache(ref), dev(table), dev([0, 60, 110], I32), dev(lens, I32)))
    assert np.isnan(got[:60]).all()
    table[0, 3] = 0
    want, tol = kv8_ref.attention(q, ref, table, np.array([0, 60, 110]), lens, None)
    assert np.all(np.abs(got[60:] - want[60:]) <= tol[60:])


@pytest.mark.parametrize("n", [3, 40])
def test_attention_rows_without_keys(n):
    """Positions before the first key (kv_len below the request's rows) give zeros, gated or not."""
    r = np.random.default_rng(n)
    got = attention_case(r, [2, 0, 50], [n, n, n], 16, 2, 128, 16)
    assert np.all(got[:n - 2] == 0) and np.all(got[n:2 * n] == 0)


@pytest.mark.parametrize("sigma", [0.0, 1e-30, 8.0, 60.0])
@pytest.mark.parametrize("n", [1, 30])
def test_attention_score_sizes(sigma, n):
    """Scores from all equal to one key far above the rest."""
    attention_case(np.random.default_rng(8), [90], [n], 16, 2, 128, 16, sigma=sigma)


@pytest.mark.parametrize("n", [2, 40])
def test_attention_scales_far_apart(n):
    """Pages of zeros (the smallest scale) and of values 2^20 apart in one row; the running reference follows both."""
    r = np.random.default_rng(n)
    page, heads, kvh, dim, total = 16, 8, 1, 64, 96
    table, pages = tables(r, [total], page)
    ref = random_cache(r, pages, kvh, page, dim)
    for j, e in enumerate((-100, 0, 20, -20, -100, 3)):
        ref.scales[1][table[0, j]] = 2.0 ** e
    ref.codes[1][table[0, 0]] = 0
    ref.scales[0][table[0, 4]] = 2.0 ** -100
    q = r.standard_normal((n, heads, dim)).astype(F32)
    got = host(ops.attn_kv8_rows(dev(q), gpu_cache(ref), dev(table), dev([0, n], I32), dev([total], I32)))
    want, tol = kv8_ref.attention(q, ref, table, [0, n], [total])
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("n", [1, 40])
def test_attention_non_finite(n):
    """A marked page shows in the rows that see it and in no others; a query row's NaN in that row alone."""
    r = np.random.default_rng(n)
    page, heads, kvh, dim = 16, 4, 2, 64
    lens = [60, 60, 45]
    table, pages = tables(r, lens, page)
    ref = random_cache(r, pages, kvh, page, dim)
    cache = gpu_cache(ref)
    cache.k_scale[int(table[0, 3]), 1] = float("nan")     # request 0, tokens 48.., KV head 1
    cache.v_scale[int(table[1, 0]), 0] = float("nan")     # request 1, every row, KV head 0
    cache.v_scale[int(table[2, 2]), 0] = float("nan")     # request 2, tokens 32.., KV head 0
    q = r.standard_normal((3 * n, heads, dim)).astype(F32)
    q[2 * n, 3, 7] = np.nan
    start = np.array([0, n, 2 * n, 3 * n], I32)
    got = host(ops.attn_kv8_rows(dev(q), cache, dev(table), dev(start), dev(lens, I32)))
    want, tol = kv8_ref.attention(q, ref, table, start, lens)
    bad = np.zeros((3 * n, heads), bool)
    for i in range(n):
        bad[i, 2:] = lens[0] - n + i >= 48
        bad[n + i, :2] = True
        bad[2 * n + i, :2] = lens[2] - n + i >= 32
    bad[2 * n, 3] = True
    assert np.all(np.isnan(got[bad]))
    assert np.all(np.abs(got[~bad] - want[~bad]) <= tol[~bad])


@pytest.mark.parametrize("n", [1, 40])
def test_attention_bad_pages_are_not_followed(n):
    """Page ids outside the cache and lengths past the table row: NaN for the rows that see them, nothing read there."""
    r = np.random.default_rng(n)
    page, heads, kvh, dim = 16, 4, 2, 64
    lens = [64, 64, 64, 64]
    table, pages = tables(r, lens, page)
    ref = random_cache(r, pages, kvh, page, dim)
    bad = table.copy()
    bad[0, 1], bad[1, 3], bad[2, 0] = pages, -1, 2 ** 31 - 1
    q = r.standard_normal((4 * n, heads, dim)).astype(F32)
    start = np.arange(5).astype(I32) * n
    got = host(ops.attn_kv8_rows(dev(q), gpu_cache(ref), dev(bad), dev(start), dev(lens[:3] + [65], I32)))
    want, tol = kv8_ref.attention(q, ref, table, start, lens)
    assert np.all(np.isnan(got[2 * n:]))
    for i in range(n):
        p = 64 - n + i
        for b, first in ((0, 16), (1, 48)):
            row = b * n + i
            if p >= first:
                assert np.all(np.isnan(got[row]))
            else:
                assert np.all(np.abs(got[row] - want[row]) <= tol[row])


def test_attention_offsets_past_32_bits():
    """Codes past 4 GiB: the last pages of a large cache, stored, read and attended."""
    page, kvh, dim = 1024, 8, 256
    pages = (5 << 30) // (page * kvh * dim)
    r = np.random.default_rng(0)
    cache = ops.Kv8Cache(torch.empty((pages, kvh, page, dim), dtype=torch.int8, device="cuda"),
                         torch.empty((pages, kvh, page // 8, dim, 8), dtype=torch.int8, device="cuda"),
                         torch.zeros((pages, kvh), device="cuda"), torch.zeros((pages, kvh), device="cuda"))
    n = 40
    slots = ((pages - 1) * page + np.arange(n)).astype(I32)
    k, v = (r.standard_normal((n, kvh, dim)).astype(F32) for _ in range(2))
    ops.kv8_store_rows(dev(k), dev(v), dev(slots), cache)
    small = kv8_ref.Cache(1, kvh, page, dim)
    small.store(0, k, np.arange(n))
    small.store(1, v, np.arange(n))
    gk, gv = (host(t) for t in ops.kv8_read_rows(cache, dev(slots)))
    assert np.array_equal(gk, small.values(0, np.arange(n)).astype(F32))
    assert np.array_equal(gv, small.values(1, np.arange(n)).astype(F32))
    for fresh in (1, n):
        q = r.standard_normal((fresh, 16, dim)).astype(F32)
        got = host(ops.attn_kv8_rows(dev(q), cache, dev([[pages - 1]], I32), dev([0, fresh], I32), dev([n], I32)))
        want, tol = kv8_ref.attention(q, small, [[0]], [0, fresh], [n])
        assert np.all(np.abs(got - want) <= tol)


# ------------------------------------------------------------------ together, graphs, streams, refusals
def test_steps_of_a_batch_in_a_graph():
    """Plan, store and attention of padded steps, captured once and replayed with other lengths and rows; every replay
    equals the eager calls bit for bit, rows behind the last request are left alone, and pages come from the list."""
    r = np.random.default_rng(11)
    page, heads, kvh, dim, requests, rows, width = 16, 8, 2, 64, 5, 24, 6
    cache, twin = (ops.kv8_cache(40, kvh, dim, page) for _ in range(2))
    free = dev(r.permutation(40), I32)
    ws = torch.empty(ops.attn_kv8_workspace_bytes(rows, requests, heads, kvh, dim), dtype=torch.uint8, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    st = {"cached": torch.zeros(requests, **i32), "fresh": torch.zeros(requests, **i32),
          "table": torch.zeros((requests, width), **i32), "head": torch.zeros(1, **i32)}
    q, gate = torch.zeros((rows, heads, dim), device="cuda"), torch.zeros((rows, heads, dim), device="cuda")
    k, v = torch.zeros((rows, kvh, dim), device="cuda"), torch.zeros((rows, kvh, dim), device="cuda")
    out = torch.zeros((rows, heads, dim), device="cuda")
    bufs = dict(row_start=torch.zeros(requests + 1, **i32), kv_len=torch.zeros(requests, **i32),
                slots=torch.zeros(rows, **i32), pos=torch.zeros(rows, **i32))

    def step(cache, table, head, out):
        ops.kv8_plan(st["cached"], st["fresh"], table, free, head, page, rows, free_head_out=head, **bufs)
        ops.kv8_store_rows(k, v, bufs["slots"], cache)
        ops.attn_kv8_rows(q, cache, table, bufs["row_start"], bufs["kv_len"], gate=gate, workspace=ws, out=out)

    step(cache, st["table"], st["head"], out)   # idle requests; loads the kernels
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(cache, st["table"], st["head"], out)
    table2, head2, out2 = st["table"].clone(), st["head"].clone(), torch.zeros_like(out)
    ref = kv8_ref.Cache(40, kvh, page, dim)
    lens = np.zeros(requests, int)
    for fresh in ([17, 1, 0, 3, 0], [1, 1, 2, 1, 0], [1, 0, 1, 1, 20], [1, 1, 1, 1, 1]):
        st["cached"].copy_(dev(lens, I32))
        st["fresh"].copy_(dev(fresh, I32))
        for t in (q, k, v, gate):
            t.copy_(dev(r.standard_normal(tuple(t.shape)).astype(F32)))
        out.fill_(3.0)
        out2.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        slots = host(bufs["slots"])
        step(twin, table2, head2, out2)
        assert torch.equal(out, out2) and torch.equal(st["table"], table2) and torch.equal(st["head"], head2)
        ref.store(0, host(k), slots)
        ref.store(1, host(v), slots)
        lens += fresh
        n = int(np.sum(fresh))
        start = np.concatenate([[0], np.cumsum(fresh)])
        want, tol = kv8_ref.attention(host(q), ref, host(st["table"]), start, lens, host(gate))
        got = host(out)
        assert np.all(np.abs(got[:n] - want[:n]) <= tol[:n])
        assert np.all(got[n:] == 3.0)


def test_attention_on_a_stream_of_its_own_repeats():
    """The same call on another stream and again: the same bits (nothing depends on the order of workgroups)."""
    r = np.random.default_rng(2)
    lens, fresh = [900, 1200, 80], [1, 3, 60]
    table, pages = tables(r, lens, 16)
    cache = gpu_cache(random_cache(r, pages, 2, 16, 128))
    q = dev(r.standard_normal((64, 8, 128)).astype(F32))
    args = (q, cache, dev(table), dev([0, 1, 4, 64], I32), dev(lens, I32))
    first = ops.attn_kv8_rows(*args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = ops.attn_kv8_rows(*args)
    other = torch.empty_like(q)
    torch.cuda.synchronize()
    ops.attn_kv8_rows(*args, out=other, stream=s)
    s.synchronize()
    assert torch.equal(first, again) and torch.equal(first, other)


def test_empty_calls_and_shapes():
    cache = ops.kv8_cache(4, 2, 64, 16)
    empty = torch.empty((0, 2, 64), device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    ops.kv8_store_rows(empty, empty, none, cache)
    assert ops.kv8_read_rows(cache, none)[0].shape == (0, 2, 64)
    q = torch.empty((0, 4, 64), device="cuda")
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    assert ops.attn_kv8_rows(q, cache, i(0).view(1, 1), i(0, 0), i(3)).shape == (0, 4, 64)
    with pytest.raises(ValueError):
        ops.kv8_store_rows(torch.empty((1, 2, 32), device="cuda"), torch.empty((1, 2, 32), device="cuda"), i(0), cache)
    with pytest.raises(ValueError):
        ops.attn_kv8_rows(torch.empty((1, 4, 64), device="cuda"), cache, i(0).view(1, 1), i(0, 1, 2), i(3))
    with pytest.raises(_lib.QwenError):
        ops.attn_kv8_rows(torch.empty((1, 3, 64), device="cuda"), cache, i(0).view(1, 1), i(0, 1), i(3))
    with pytest.raises(_lib.QwenError, match="workspace"):
        ops.attn_kv8_rows(torch.empty((1, 4, 64), device="cuda"), cache, i(0).view(1, 1), i(0, 1), i(3),
                          workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))
