"""The paged 4-bit cache: storing and reading rows, attention of several requests' rows over it.

Codes, scales and minima are compared exactly (they do not depend on how a quotient is evaluated), attention with the
tolerance that tests/kv4_ref.py derives from its roundings."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import kv4_ref
from qwen35_hip import _lib, ops

pytestmark = pytest.mark.gpu
F32, I32 = np.float32, np.int32
NAMES = ("k", "v", "k_scale", "k_min", "v_scale", "v_min")


def dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).cuda()


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


def bits(t):
    return host(t.view(torch.int16)).view(np.uint16) if t.dtype == torch.bfloat16 else host(t)


def gpu_cache(ref):
    return ops.Kv4Cache(*(dev(a.view(np.int16)).view(torch.bfloat16) if a.dtype == np.uint16 else dev(a)
                          for a in ref.arrays()))


def random_cache(r, pages, heads, page, dim):
    ref = kv4_ref.Cache(pages, heads, page, dim)
    for w in (0, 1):
        ref.codes[w] = r.integers(0, 16, ref.codes[w].shape).astype(np.float64)
        ref.scale[w] = kv4_ref.bf16_up(0.15 * 2.0 ** r.uniform(-3, 1, ref.scale[w].shape)).astype(np.float64)
        ref.low[w] = kv4_ref.bf16_down((-8 * ref.scale[w] * r.uniform(0.5, 1.5, ref.low[w].shape)).astype(F32)).astype(np.float64)
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


def same_cache(cache, ref, only=None):
    """Every array of the cache, bit for bit; NaN scales as NaNs. `only`: slots that are looked at."""
    for name, want in zip(NAMES, ref.arrays()):
        got = bits(getattr(cache, name))
        if only is not None and name != "k_scale":
            p, o = np.asarray(only) // ref.page, np.asarray(only) % ref.page
            if name == "v":
                sh = (4 * (o % 8 // 2 + 4 * (o % 2)))[:, None, None]
                got, want = (((a.view(np.uint32)[..., 0][p, :, o // 8] >> sh) & 15) for a in (got, want))
            else:
                got, want = got[p, :, o], want[p, :, o]
        elif only is not None:
            p, o = np.asarray(only) // ref.page, np.asarray(only) % ref.page
            got, want = got[p, :, o // 8, :, o % 8], want[p, :, o // 8, :, o % 8]
        if name.endswith("scale"):
            nan = (want & 0x7fff) > 0x7f80
            assert np.array_equal((got & 0x7fff) > 0x7f80, nan), name
            got, want = np.where(nan, 0, got), np.where(nan, 0, want)
        assert np.array_equal(got, want), name


def varied(r, n, heads, dim):
    """Rows whose sizes vary by powers of ten, some of them far from zero."""
    x = r.standard_normal((n, heads, dim)) * 10.0 ** r.integers(-3, 3, (n, heads, 1))
    return (x + 10.0 ** r.uniform(-3, 3, (n, heads, 1)) * r.integers(-1, 2, (n, heads, 1))).astype(F32)


# ------------------------------------------------------------------ store, read
@pytest.mark.parametrize("page,heads,dim", [(8, 1, 64), (16, 2, 256), (64, 2, 256), (32, 5, 128), (1024, 3, 64)])
def test_store_in_steps(page, heads, dim):
    """Requests filled by steps of 1 to 2 pages + 3 tokens, rows without a slot between: all arrays, untouched parts too."""
    r = np.random.default_rng(page + dim)
    steps = [[1, 3, 0, 2 * page + 3], [1, page - 1, 5, 1], [1, 1, 1, 1], [page, 2, 7, 1], [1, 1, page + 1, 9]]
    table, pages = tables(r, np.sum(steps, axis=0), page)
    ref = random_cache(r, pages, heads, page, dim)
    cache = gpu_cache(ref)
    at = np.zeros(4, int)
    for fresh in steps:
        slots = np.concatenate([[-1]] + [table[b][t // page] * page + t % page for b in range(4)
                                         for t in [np.arange(at[b], at[b] + fresh[b])]] + [[-7]]).astype(I32)
        k, v = varied(r, len(slots), heads, dim), varied(r, len(slots), heads, dim)
        ops.kv4_store_rows(dev(k), dev(v), dev(slots), cache)
        ref.store(0, k, slots)
        ref.store(1, v, slots)
        at += fresh
        same_cache(cache, ref)
    live = np.concatenate([table[b][t // page] * page + t % page for b in range(4) for t in [np.arange(at[b])]])
    read = np.concatenate([live, [-1]]).astype(I32)
    for w, got in enumerate(host(t) for t in ops.kv4_read_rows(cache, dev(read))):
        assert np.array_equal(got[:-1], ref.values(w, live).astype(F32))
        assert np.all(got[-1] == 0)


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 15, 16, 17, 64, 1023, 2500])
@pytest.mark.parametrize("first", [0, 37])
def test_store_long_runs(rows, first):
    r = np.random.default_rng(rows)
    page, heads, dim = 128, 2, 64
    table, pages = tables(r, [rows + first], page)
    ref = random_cache(r, pages, heads, page, dim)
    cache = gpu_cache(ref)
    t = np.arange(first, first + rows)
    slots = (table[0][t // page] * page + t % page).astype(I32)
    k, v = varied(r, rows, heads, dim), varied(r, rows, heads, dim)
    ops.kv4_store_rows(dev(k), dev(v), dev(slots), cache)
    ref.store(0, k, slots)
    ref.store(1, v, slots)
    same_cache(cache, ref)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("order", ["shuffled", "falling", "every third"])
def test_store_in_any_order(order, dim):
    """Slots of one octet of tokens from rows far apart: no row takes another one's nibble."""
    r = np.random.default_rng(dim)
    page, heads, pages = 32, 3, 7
    slots = {"shuffled": r.permutation(pages * page)[:190], "falling": np.arange(pages * page - 3, 11, -1),
             "every third": np.concatenate([np.arange(2, pages * page, 3), np.arange(0, pages * page, 3)])}[order].astype(I32)
    ref = random_cache(r, pages, heads, page, dim)
    cache = gpu_cache(ref)
    k, v = varied(r, len(slots), heads, dim), varied(r, len(slots), heads, dim)
    ops.kv4_store_rows(dev(k), dev(v), dev(slots), cache)
    ref.store(0, k, slots)
    ref.store(1, v, slots)
    same_cache(cache, ref)


def test_store_ties_and_borders():
    """Quotients on and next to half steps: the nearest code, ties to even, by the 64-bit quotient."""
    page, dim = 8, 64
    ref = kv4_ref.Cache(4, 1, page, dim)
    cache = gpu_cache(ref)
    rows = []
    for low, scale in ((0.0, 1.0), (-7.5, 1.0), (-8.0, 1.0), (0.25, 0.375), (-3.0, 0.0078125), (1.0, 1.0078125)):
        half = low + scale * (np.arange(15) + 0.5)
        for near in (half, np.nextafter(half.astype(F32), F32(99)), np.nextafter(half.astype(F32), F32(-99))):
            x = np.full(dim, low, F32)
            x[1:16] = near
            x[16] = low + 15 * scale
            x[17:33] = low + scale * np.arange(16)
            rows.append(x)
    x = np.stack(rows)[:, None]
    slots = np.arange(len(x), dtype=I32)
    ops.kv4_store_rows(dev(x), dev(-x), dev(slots), cache)
    ref.store(0, x, slots)
    ref.store(1, -x, slots)
    same_cache(cache, ref)


@pytest.mark.parametrize("size", [0.0, 1e-45, 1e-38, 1e-30, 1e-10, 1e30, 1.6e38])
def test_store_extreme_sizes(size):
    ref = kv4_ref.Cache(1, 2, 16, 64)
    cache = gpu_cache(ref)
    r = np.random.default_rng(1)
    x = (r.uniform(-1, 1, (5, 2, 64)) * size).astype(F32)
    x[3] = np.abs(x[3])
    x[4] = F32(size) * F32(0.7)   # all the same
    ops.kv4_store_rows(dev(x), dev(-x), dev(np.arange(5), I32), cache)
    ref.store(0, x, np.arange(5))
    ref.store(1, -x, np.arange(5))
    same_cache(cache, ref)
    for w, got in enumerate(host(t) for t in ops.kv4_read_rows(cache, dev(np.arange(5), I32))):
        assert np.array_equal(got, ref.values(w, np.arange(5)).astype(F32))
        assert np.all(np.abs(got - (x, -x)[w]) <= 0.51 * np.repeat(ref.scale[w][0, :, :5].swapaxes(0, 1), 64, -1))


def test_store_non_finite():
    """An infinity or NaN marks its group alone: 64 keys, or a token's values of a head."""
    ref = kv4_ref.Cache(2, 2, 8, 128)
    cache = gpu_cache(ref)
    x = np.random.default_rng(0).standard_normal((6, 2, 128)).astype(F32)
    x[1, 1, 5], x[2, 0, 70], x[3, 0, 0], x[4, 1, 127] = np.inf, np.nan, -np.inf, -3.4e38
    slots = np.arange(3, 9, dtype=I32)
    ops.kv4_store_rows(dev(x), dev(x), dev(slots), cache)
    ref.store(0, x, slots)
    ref.store(1, x, slots)
    same_cache(cache, ref)
    k, v = (host(t) for t in ops.kv4_read_rows(cache, dev(slots)))
    want = np.zeros((6, 2, 2), bool)
    want[1, 1, 0] = want[2, 0, 1] = want[3, 0, 0] = want[4, 1, 1] = True
    assert np.array_equal(np.isnan(k), np.repeat(want, 64, -1))
    assert np.array_equal(np.isnan(v), np.repeat(want.any(-1, keepdims=True), 128, -1))
    x = np.abs(x[:1])
    ops.kv4_store_rows(dev(x), dev(x), dev(slots[2:3]), cache)   # stored again: as new
    assert not np.isnan(host(ops.kv4_read_rows(cache, dev(slots[2:3]))[0])).any()


def test_store_strided_unaligned_and_out_of_cache():
    r = np.random.default_rng(5)
    page, heads, dim, rows = 16, 2, 64, 21
    ref = random_cache(r, 3, heads, page, dim)
    cache = gpu_cache(ref)
    w = dev(r.standard_normal((rows, 3 * heads * dim + 3)).astype(F32))
    for off in (0, 1):   # 16-byte aligned rows are not the only ones
        kt = w[:, off:off + heads * dim].view(rows, heads, dim)
        vt = w[:, off + 2 * heads * dim:off + 3 * heads * dim].view(rows, heads, dim)
        slots = np.concatenate([np.arange(5, 5 + rows - 3), [48, 2 ** 31 - 1, -1]]).astype(I32)
        ops.kv4_store_rows(kt, vt, dev(slots), cache)
        ref.store(0, host(kt), slots)
        ref.store(1, host(vt), slots)
        same_cache(cache, ref)
        got = host(ops.kv4_read_rows(cache, dev(slots))[1])
        assert np.all(np.isnan(got[rows - 3:rows - 1])) and np.all(got[rows - 1] == 0)


def test_store_one_slot_twice_stays_in_it():
    """What two rows of one slot leave there is not defined; every other slot is as it was or as its row says."""
    r = np.random.default_rng(9)
    page, heads, dim = 16, 2, 128
    ref = random_cache(r, 3, heads, page, dim)
    cache = gpu_cache(ref)
    slots = np.array([3, 4, 4, 5, 20, 3, 21], I32)
    x = r.standard_normal((7, heads, dim)).astype(F32)
    ops.kv4_store_rows(dev(x), dev(x), dev(slots), cache)
    ref.store(0, x, slots)
    ref.store(1, x, slots)
    same_cache(cache, ref, only=[s for s in range(3 * page) if s not in (3, 4)])


# ------------------------------------------------------------------ attention
def attention_case(r, lens, fresh, heads, kvh, dim, page, gated=True, pad=0, sigma=1.0, width=None):
    table, pages = tables(r, lens, page, width)
    ref = random_cache(r, pages, kvh, page, dim)
    rows = int(np.sum(fresh))
    start = np.concatenate([[0], np.cumsum(fresh)]).astype(I32)
    q = (sigma * r.standard_normal((rows + pad, heads, dim))).astype(F32)
    gate = r.standard_normal((rows + pad, heads, dim)).astype(F32) if gated else None
    out = torch.full((rows + pad, heads, dim), 7.0, device="cuda")
    got = host(ops.attn_kv4_rows(dev(q), gpu_cache(ref), dev(table), dev(start), dev(lens, I32),
                                 gate=None if gate is None else dev(gate), out=out))
    want, tol = kv4_ref.attention(q, ref, table, start, lens, gate)
    close(got, want, tol)
    return got


def close(got, want, tol):
    err = np.abs(got - want)
    assert np.all(err <= tol), (float((err / np.maximum(tol, 1e-300)).max()), np.argwhere(~(err <= tol))[0])


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
    """From few rows to many, behind a cached prefix and without one."""
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
    attention_case(r, [2600, 1300], [1, 1], 8, 1, 256, 16)


@pytest.mark.parametrize("heads,kvh,dim,page", [(16, 2, 256, 64), (6, 2, 64, 8), (8, 8, 128, 16)])
def test_attention_prompts_in_pieces(heads, kvh, dim, page):
    """Chunks of prompts behind long prefixes: too few row tiles for the card, so that their keys are cut and joined.
    Lengths around the pieces' and tiles' ends; two chunks whose pieces differ in number; single tokens beside them."""
    r = np.random.default_rng(dim)
    for n, before in ((40, 473), (33, 991), (70, 1500), (36, 220)):
        attention_case(r, [before + n], [n], heads, kvh, dim, page, gated=n != 33)
    attention_case(r, [1100, 900, 530, 64], [50, 1, 35, 40], heads, kvh, dim, page, pad=2)


@pytest.mark.parametrize("lens,fresh,heads,kvh", [
    ([70 + i for i in range(30)], [70] * 30, 16, 2),   # more row tiles than CUs, each short
    ([1000], [1000], 32, 1),                           # nearly as many as CUs, of 1 to 32 tiles
    ([500, 1, 0, 1700], [400, 1, 0, 600], 32, 1),
    ([40] * 60, [40] * 60, 16, 2),
])
def test_attention_prompts_as_a_line(lens, fresh, heads, kvh):
    """Calls whose row tiles and KV heads are cut as one line of tiles: workgroups with the ends and the beginnings of several."""
    r = np.random.default_rng(len(lens) + heads)
    attention_case(r, lens, fresh, heads, kvh, 64, 32, gated=len(lens) > 1, pad=1)


@pytest.mark.parametrize("heads,kvh,dim,page,n,total", [(40, 2, 64, 8, 210, 510), (48, 2, 128, 16, 345, 500),
                                                        (64, 2, 256, 64, 260, 400), (64, 8, 64, 16, 130, 200)])
def test_attention_chunks_of_many_units(heads, kvh, dim, page, n, total):
    """A chunk whose row tiles are cut in pieces, in each head dim; and one of more blocks of 8 pairs than the card has places for
    workgroups of few rows, but few enough for them. Single tokens beside them."""
    r = np.random.default_rng(dim + heads)
    attention_case(r, [total, 77, total // 2], [n, 1, 1], heads, kvh, dim, page, pad=1)


@pytest.mark.parametrize("heads,kvh,dim,page", [(16, 2, 256, 64), (6, 2, 64, 8), (8, 8, 128, 16)])
def test_attention_light_calls_of_long_tables(heads, kvh, dim, page):
    """Tables that could hold long contexts, so that the lengths alone say how much a call is: rows of one request and of several,
    prompts short and long beside single tokens, more than 256 requests."""
    r = np.random.default_rng(dim + 1)
    for lens, fresh in (([41 + 17], [17]), ([33, 900, 60, 1], [33, 12, 30, 1]), ([130, 700], [100, 9]), ([20] * 300, [0, 9, 1] * 100)):
        attention_case(r, lens, fresh, heads, kvh, dim, page, pad=2, width=70000 // page)


def test_attention_gate_sizes():
    """Gates to where e^-x and e^x leave the range of fp32; below it results are subnormal numbers, as near as their step."""
    r = np.random.default_rng(17)
    for n in (1, 40):
        lens = np.array([n + 20])
        table, pages = tables(r, lens, 16)
        ref = random_cache(r, pages, 2, 16, 64)
        start = np.array([0, n], I32)
        q = r.standard_normal((n, 8, 64)).astype(F32)
        gate = r.choice(np.array([-200, -104, -100, -95, -90, -88, -87, -81, -80, -79, -1, 0, 60, 90, 200], F32), (n, 8, 64))
        got = host(ops.attn_kv4_rows(dev(q), gpu_cache(ref), dev(table), dev(start), dev(lens, I32), gate=dev(gate)))
        want, tol = kv4_ref.attention(q, ref, table, start, lens, gate)
        close(got, want, tol + 2.0 ** -147)   # two roundings to subnormal numbers


def test_attention_no_more_rows_than_requests():
    """A batch padded to many requests, one of which has most of the rows."""
    r = np.random.default_rng(33)
    attention_case(r, [700, 0, 90, 1] + [0] * 60, [58, 0, 5, 1] + [0] * 60, 16, 2, 128, 16)
    attention_case(r, [0] * 79 + [130], [0] * 79 + [80], 8, 2, 64, 8, pad=0)


@pytest.mark.parametrize("n", [1, 70])
def test_attention_many_requests(n):
    """More requests than a wave has lanes, most of them idle or short."""
    r = np.random.default_rng(n)
    lens = r.integers(0, 40, 150)
    fresh = np.minimum(lens, r.integers(0, 3, 150))
    lens[130] += 300
    fresh[130] = n
    attention_case(r, lens.tolist(), fresh.tolist(), 8, 2, 64, 16)


def test_attention_rows_of_a_part_of_a_step():
    """row_start need not begin at 0 nor end at the last row: the rows outside are left as they were."""
    r = np.random.default_rng(6)
    page, heads, kvh, dim, lens = 16, 8, 2, 64, [100, 37]
    table, pages = tables(r, lens, page)
    ref = random_cache(r, pages, kvh, page, dim)
    for n in (1, 45):
        q = r.standard_normal((2 * n + 6, heads, dim)).astype(F32)
        start = np.array([2, 2 + n, 2 + 2 * n])
        out = torch.full(q.shape, 5.0, device="cuda")
        got = host(ops.attn_kv4_rows(dev(q), gpu_cache(ref), dev(table), dev(start, I32), dev(lens, I32), out=out))
        want, tol = kv4_ref.attention(q, ref, table, start, lens)
        close(got[2:2 + 2 * n], want[2:2 + 2 * n], tol[2:2 + 2 * n])
        assert np.all(got[:2] == 5.0) and np.all(got[2 + 2 * n:] == 5.0)


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
    """Tokens of zeros (the smallest scale), of one value, and of values 2^20 apart, among 8 neighbours and across tiles; the
    running reference follows them."""
    r = np.random.default_rng(n)
    page, heads, kvh, dim, total = 16, 8, 1, 64, 96
    table, pages = tables(r, [total], page)
    ref = random_cache(r, pages, kvh, page, dim)
    for t in range(total):
        at = np.s_[table[0, t // page], :, t % page]
        e = (-100, 0, 20, -20, 3, -100, 0)[(t // 40 * 3 + t) % 7]
        ref.scale[1][at] = 2.0 ** e
        ref.low[1][at] = -(2.0 ** e) * 7
        if e == -100:
            ref.codes[1][at] = 0
            ref.low[1][at] = 0.0 if t % 2 else 1.5 * 2.0 ** 10
    ref.scale[0][table[0, 4]] = 2.0 ** -100
    q = r.standard_normal((n, heads, dim)).astype(F32)
    got = host(ops.attn_kv4_rows(dev(q), gpu_cache(ref), dev(table), dev([0, n], I32), dev([total], I32)))
    want, tol = kv4_ref.attention(q, ref, table, [0, n], [total])
    close(got, want, tol)


@pytest.mark.parametrize("keys,values", [(0, 96), (0, 40), (0, -44), (0, -90), (96, 0), (-90, 0)])
@pytest.mark.parametrize("n", [1, 40])
def test_attention_sizes(n, keys, values):
    """Keys and values of sizes to both ends of what is held, queries of the keys' inverse size."""
    r = np.random.default_rng(keys + 2 * values + n + 500)
    page, heads, kvh, dim, total = 16, 8, 2, 128, 700
    table, pages = tables(r, [total], page)
    ref = random_cache(r, pages, kvh, page, dim)
    for w, e in ((0, keys), (1, values)):
        ref.scale[w] *= 2.0 ** e
        ref.low[w] *= 2.0 ** e
    q = (2.0 ** -keys * r.standard_normal((n, heads, dim))).astype(F32)
    got = host(ops.attn_kv4_rows(dev(q), gpu_cache(ref), dev(table), dev([0, n], I32), dev([total], I32)))
    want, tol = kv4_ref.attention(q, ref, table, [0, n], [total])
    close(got, want, tol)


def test_attention_zeros_before_values():
    """Tokens of zeros keep their weight in the sum when larger values come behind them, in any tile."""
    r = np.random.default_rng(1)
    page, heads, kvh, dim, total = 64, 8, 1, 128, 640
    table, pages = tables(r, [total], page)
    ref = random_cache(r, pages, kvh, page, dim)
    for t in range(600):
        at = np.s_[table[0, t // page], :, t % page]
        ref.scale[1][at], ref.low[1][at], ref.codes[1][at] = 2.0 ** -100, 0.0, 0
    for t in range(600, total):
        at = np.s_[table[0, t // page], :, t % page]
        ref.scale[1][at], ref.low[1][at] = 2.0 ** 30, -(2.0 ** 33)
    for n in (1, 36):
        q = 0.1 * r.standard_normal((n, heads, dim)).astype(F32)
        got = host(ops.attn_kv4_rows(dev(q), gpu_cache(ref), dev(table), dev([0, n], I32), dev([total], I32)))
        want, tol = kv4_ref.attention(q, ref, table, [0, n], [total])
        close(got, want, tol)


@pytest.mark.parametrize("n", [1, 40])
def test_attention_non_finite(n):
    """A marked group shows in the rows that see its token and in no others; a query row's NaN in that row alone."""
    r = np.random.default_rng(n)
    page, heads, kvh, dim = 16, 4, 2, 128
    lens = [60, 60, 45]
    table, pages = tables(r, lens, page)
    ref = random_cache(r, pages, kvh, page, dim)
    cache = gpu_cache(ref)
    cache.k_scale[int(table[0, 3]), 1, 0, 1, 3] = float("nan")     # request 0, token 51, KV head 1
    cache.v_scale[int(table[1, 0]), 0, 2] = float("nan")           # request 1, token 2, KV head 0
    cache.v_min[int(table[2, 2]), 0, 5] = float("nan")             # request 2, token 37, KV head 0
    cache.k_min[int(table[2, 2]), 1, 4, 0] = float("inf")          # request 2, token 36, KV head 1: a score without value
    q = r.standard_normal((3 * n, heads, dim)).astype(F32)
    q[2 * n, 3, 7] = np.nan
    start = np.array([0, n, 2 * n, 3 * n], I32)
    got = host(ops.attn_kv4_rows(dev(q), cache, dev(table), dev(start), dev(lens, I32)))
    want, tol = kv4_ref.attention(q, ref, table, start, lens)
    bad = np.zeros((3 * n, heads), bool)
    skip = np.zeros((3 * n, heads), bool)
    for i in range(n):
        bad[i, 2:] = lens[0] - n + i >= 51
        bad[n + i, :2] = lens[1] - n + i >= 2
        bad[2 * n + i, :2] = lens[2] - n + i >= 37
        skip[2 * n + i, 2:] = lens[2] - n + i >= 36   # infinite keys: whatever inf - inf gives
    bad[2 * n, 3] = True
    assert np.all(np.isnan(got[bad]))
    rest = ~bad & ~skip
    close(got[rest], want[rest], tol[rest])


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
    got = host(ops.attn_kv4_rows(dev(q), gpu_cache(ref), dev(bad), dev(start), dev(lens[:3] + [65], I32)))
    want, tol = kv4_ref.attention(q, ref, table, start, lens)
    assert np.all(np.isnan(got[2 * n:]))
    for i in range(n):
        p = 64 - n + i
        for b, first in ((0, 16), (1, 48)):
            row = b * n + i
            if p >= first:
                assert np.all(np.isnan(got[row]))
            else:
                close(got[row], want[row], tol[row])


def test_attention_prompts_in_pieces_bad_page():
    """A page outside the cache makes every row of its request NaN that sees it, whichever piece holds it."""
    r = np.random.default_rng(31)
    lens, fresh = [900, 700], [60, 50]
    table, pages = tables(r, lens, 32)
    table[0, 3] = pages + 5
    ref = random_cache(r, pages, 2, 32, 128)
    q = r.standard_normal((110, 16, 128)).astype(F32)
    got = host(ops.attn_kv4_rows(dev(q), gpu_cache(ref), dev(table), dev([0, 60, 110], I32), dev(lens, I32)))
    assert np.isnan(got[:60]).all()
    table[0, 3] = 0
    want, tol = kv4_ref.attention(q, ref, table, np.array([0, 60, 110]), lens, None)
    close(got[60:], want[60:], tol[60:])


def test_attention_odd_starts_stay_in_bounds():
    """row_start that falls or leaves the step, negative and too large lengths: rows that belong to one request alone are
    right, and the padding behind `out` is untouched."""
    r = np.random.default_rng(12)
    page, heads, kvh, dim = 16, 4, 2, 64
    table, pages = tables(r, [64] * 4, page)
    ref = random_cache(r, pages, kvh, page, dim)
    q = dev(r.standard_normal((12, heads, dim)).astype(F32))
    for start, lens in (([0, 5, 3, 99, 4], [64, 64, 64, 64]), ([-7, 3, 6, 2 ** 31 - 1, 2 ** 31 - 1], [64, -5, 64, 1000]),
                        ([2 ** 31 - 1, 0, 0, 0, 0], [1, 2, 3, 4])):
        buf = torch.full((20, heads, dim), 3.0, device="cuda")
        ops.attn_kv4_rows(q, gpu_cache(ref), dev(table), dev(start, I32), dev(lens, I32), out=buf[4:16])
        torch.cuda.synchronize()
        assert (buf[:4] == 3.0).all() and (buf[16:] == 3.0).all()


def test_offsets_past_32_bits():
    """Codes past 4 GiB: the last pages of a large cache, stored, read and attended."""
    page, kvh, dim = 1024, 8, 256
    pages = (5 << 30) // (page * kvh * dim // 2)
    r = np.random.default_rng(0)
    cache = ops.kv4_cache(pages, kvh, dim, page)
    n = 40
    slots = ((pages - 1) * page + np.arange(n)).astype(I32)
    k, v = (r.standard_normal((n, kvh, dim)).astype(F32) for _ in range(2))
    ops.kv4_store_rows(dev(k), dev(v), dev(slots), cache)
    small = kv4_ref.Cache(1, kvh, page, dim)
    small.store(0, k, np.arange(n))
    small.store(1, v, np.arange(n))
    gk, gv = (host(t) for t in ops.kv4_read_rows(cache, dev(slots)))
    assert np.array_equal(gk, small.values(0, np.arange(n)).astype(F32))
    assert np.array_equal(gv, small.values(1, np.arange(n)).astype(F32))
    for fresh in (1, n):
        q = r.standard_normal((fresh, 16, dim)).astype(F32)
        got = host(ops.attn_kv4_rows(dev(q), cache, dev([[pages - 1]], I32), dev([0, fresh], I32), dev([n], I32)))
        want, tol = kv4_ref.attention(q, small, [[0]], [0, fresh], [n])
        close(got, want, tol)


# ------------------------------------------------------------------ together, graphs, streams
def test_steps_of_a_batch_in_a_graph():
    """Plan, rotation, store and attention of padded steps, captured once and replayed with other lengths and rows; every
    replay equals the eager calls bit for bit, rows behind the last request are left alone, and pages come from the list."""
    r = np.random.default_rng(11)
    page, heads, kvh, dim, requests, rows, width = 16, 8, 2, 64, 5, 24, 6
    cache, twin = (ops.kv4_cache(40, kvh, dim, page) for _ in range(2))
    free = dev(r.permutation(40), I32)
    ws = torch.empty(ops.attn_kv4_workspace_bytes(rows, requests, heads, kvh, dim), dtype=torch.uint8, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    st = {"cached": torch.zeros(requests, **i32), "fresh": torch.zeros(requests, **i32),
          "table": torch.zeros((requests, width), **i32), "head": torch.zeros(1, **i32)}
    names = ("q", "k", "v", "gate")
    x = {n: torch.zeros((rows, kvh if n in "kv" else heads, dim), device="cuda") for n in names}
    work = {n: torch.zeros_like(x[n]) for n in "qk"}
    w = dev(r.uniform(0.5, 2, dim).astype(F32))
    pos3 = torch.zeros((3, rows), **i32)
    out = torch.zeros((rows, heads, dim), device="cuda")
    bufs = dict(row_start=torch.zeros(requests + 1, **i32), kv_len=torch.zeros(requests, **i32),
                slots=torch.zeros(rows, **i32), pos=torch.zeros(rows, **i32))

    def step(cache, table, head, out):
        ops.kv8_plan(st["cached"], st["fresh"], table, free, head, page, rows, free_head_out=head, **bufs)
        for n in "qk":
            work[n].copy_(x[n])
        ops.attn_qk_norm_mrope_rows(work["q"], work["k"], w, w, pos3, (16, 8, 8))
        ops.kv4_store_rows(work["k"], x["v"], bufs["slots"], cache)
        ops.attn_kv4_rows(work["q"], cache, table, bufs["row_start"], bufs["kv_len"], gate=x["gate"], workspace=ws, out=out)

    step(cache, st["table"], st["head"], out)   # idle requests; loads the kernels
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(cache, st["table"], st["head"], out)
    table2, head2, out2 = st["table"].clone(), st["head"].clone(), torch.zeros_like(out)
    ref = kv4_ref.Cache(40, kvh, page, dim)
    lens = np.zeros(requests, int)
    for fresh in ([17, 1, 0, 3, 0], [1, 1, 2, 1, 0], [1, 0, 1, 1, 20], [1, 1, 1, 1, 1]):
        st["cached"].copy_(dev(lens, I32))
        st["fresh"].copy_(dev(fresh, I32))
        for t in x.values():
            t.copy_(dev(r.standard_normal(tuple(t.shape)).astype(F32)))
        pos3.copy_(dev(r.integers(0, 50000, (3, rows)), I32))
        out.fill_(3.0)
        out2.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        slots, qr, kr = host(bufs["slots"]), host(work["q"]), host(work["k"])
        step(twin, table2, head2, out2)
        assert torch.equal(out, out2) and torch.equal(st["table"], table2) and torch.equal(st["head"], head2)
        ref.store(0, kr, slots)
        ref.store(1, host(x["v"]), slots)
        lens += fresh
        n = int(np.sum(fresh))
        start = np.concatenate([[0], np.cumsum(fresh)])
        want, tol = kv4_ref.attention(qr, ref, host(st["table"]), start, lens, host(x["gate"]))
        got = host(out)
        close(got[:n], want[:n], tol[:n])
        assert np.all(got[n:] == 3.0)


def test_attention_on_a_stream_of_its_own_repeats():
    """The same call on another stream and again: the same bits (nothing depends on the order of workgroups)."""
    r = np.random.default_rng(2)
    lens, fresh = [900, 1200, 80], [1, 3, 60]
    table, pages = tables(r, lens, 16)
    cache = gpu_cache(random_cache(r, pages, 2, 16, 128))
    q = dev(r.standard_normal((64, 8, 128)).astype(F32))
    args = (q, cache, dev(table), dev([0, 1, 4, 64], I32), dev(lens, I32))
    first = ops.attn_kv4_rows(*args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = ops.attn_kv4_rows(*args)
    other = torch.empty_like(q)
    torch.cuda.synchronize()
    ops.attn_kv4_rows(*args, out=other, stream=s)
    s.synchronize()
    assert torch.equal(first, again) and torch.equal(first, other)


def test_a_workspace_serves_fewer_rows_and_requests():
    """One sized for some rows and requests, full of the last call's numbers, serves a smaller call."""
    r = np.random.default_rng(21)
    page, heads, kvh, dim = 16, 16, 2, 128
    ws = torch.full((ops.attn_kv4_workspace_bytes(90, 8, heads, kvh, dim),), 0x7f, dtype=torch.uint8, device="cuda")
    for lens, fresh in (([400, 900, 77], [20, 1, 60]), ([1500], [1]), ([64, 300], [2, 33]), ([700] * 8, [1] * 8)):
        table, pages = tables(r, lens, page)
        ref = random_cache(r, pages, kvh, page, dim)
        start = np.concatenate([[0], np.cumsum(fresh)]).astype(I32)
        q = r.standard_normal((start[-1], heads, dim)).astype(F32)
        assert ops.attn_kv4_workspace_bytes(len(q), len(lens), heads, kvh, dim) <= ws.numel()
        got = host(ops.attn_kv4_rows(dev(q), gpu_cache(ref), dev(table), dev(start), dev(lens, I32), workspace=ws))
        close(got, *kv4_ref.attention(q, ref, table, start, lens))


@pytest.mark.parametrize("lens,fresh,heads,kvh,dim", [
    ([9000], [1], 16, 2, 256), ([700] * 150, [1] * 150, 16, 2, 128), ([300, 41], [30, 9], 16, 2, 64), ([1200, 5], [1000, 1], 16, 2, 256),
    ([90 + i for i in range(40)], [90] * 40, 16, 2, 64), ([900, 800], [900, 700], 32, 4, 128), ([4000] * 3, [12, 1, 300], 24, 8, 128)])
def test_workspace_ends_where_the_query_says(lens, fresh, heads, kvh, dim):
    """Calls that cut their keys in every way leave what lies behind the workspace as it was."""
    r = np.random.default_rng(dim)
    table, pages = tables(r, lens, 64)
    cache = ops.kv4_cache(pages, kvh, dim, 64)
    rows = int(np.sum(fresh))
    need = ops.attn_kv4_workspace_bytes(rows, len(lens), heads, kvh, dim)
    memory = torch.full((need + (1 << 20),), 0x5a, dtype=torch.uint8, device="cuda")
    q = dev(r.standard_normal((rows, heads, dim)).astype(F32))
    start = np.concatenate([[0], np.cumsum(fresh)])
    out = ops.attn_kv4_rows(q, cache, dev(table), dev(start, I32), dev(lens, I32), workspace=memory[:need])
    assert bool((out == 0).all()) and bool((memory[need:] == 0x5a).all())   # a cache of zeros


def test_gate_in_place():
    r = np.random.default_rng(14)
    table, pages = tables(r, [50, 90], 16)
    cache = gpu_cache(random_cache(r, pages, 2, 16, 64))
    q, gate = (dev(r.standard_normal((41, 4, 64)).astype(F32)) for _ in range(2))
    args = (q, cache, dev(table), dev([0, 1, 41], I32), dev([50, 90], I32))
    want = ops.attn_kv4_rows(*args, gate=gate)
    assert torch.equal(ops.attn_kv4_rows(*args, gate=gate, out=gate), want)


def test_empty_calls_and_shapes():
    cache = ops.kv4_cache(4, 2, 64, 16)
    empty = torch.empty((0, 2, 64), device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    ops.kv4_store_rows(empty, empty, none, cache)
    assert ops.kv4_read_rows(cache, none)[0].shape == (0, 2, 64)
    q = torch.empty((0, 4, 64), device="cuda")
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    assert ops.attn_kv4_rows(q, cache, i(0).view(1, 1), i(0, 0), i(3)).shape == (0, 4, 64)
    with pytest.raises(ValueError):
        ops.kv4_store_rows(torch.empty((1, 2, 32), device="cuda"), torch.empty((1, 2, 32), device="cuda"), i(0), cache)
    with pytest.raises(ValueError):
        ops.attn_kv4_rows(torch.empty((1, 4, 64), device="cuda"), cache, i(0).view(1, 1), i(0, 1, 2), i(3))
    with pytest.raises(_lib.QwenError):
        ops.attn_kv4_rows(torch.empty((1, 3, 64), device="cuda"), cache, i(0).view(1, 1), i(0, 1), i(3))
    with pytest.raises(_lib.QwenError, match="workspace"):
        ops.attn_kv4_rows(torch.empty((1, 4, 64), device="cuda"), cache, i(0).view(1, 1), i(0, 1), i(3),
                          workspace=torch.empty(0, dtype=torch.uint8, device="cuda"))
    with pytest.raises(AttributeError):   # it stays over the tensors it was made of
        cache.k = cache.k.clone()
    with pytest.raises(ValueError, match="shape"):
        ops.Kv4Cache(cache.k, cache.v, cache.k_scale, cache.v_min, cache.v_scale, cache.v_min)
    eight = ops.kv8_cache(4, 2, 64, 16)
    x, q = torch.zeros((1, 2, 64), device="cuda"), torch.zeros((1, 4, 64), device="cuda")
    for c, calls in ((cache, (ops.kv8_store_rows, ops.kv8_read_rows, ops.attn_kv8_rows)),
                     (eight, (ops.kv4_store_rows, ops.kv4_read_rows, ops.attn_kv4_rows))):
        for call, args in zip(calls, ((x, x, i(0), c), (c, i(0)), (q, c, i(0).view(1, 1), i(0, 1), i(3)))):
            with pytest.raises(ValueError, match="expected a Kv"):
                call(*args)
