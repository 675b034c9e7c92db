"""Attention over the paged 8-bit cache where its kernels meet their ends: calls with more row tiles than the card takes at
once, joins of every form, rows that belong to no request, pages of zeros beside others.

The reference is tests/kv8_ref.py's in 64 bits, a request at a time. Its tolerance stands there; here |v - out| in it is
replaced by |v| + |out|, which needs no array of rows x keys x dims and is never smaller."""

from __future__ import annotations

import kv8_ref
import numpy as np
import pytest
import torch

from qwen35_hip import ops

pytestmark = pytest.mark.gpu
F32, F64, I32 = np.float32, np.float64, np.int32


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
        ref.codes[w] = r.integers(-127, 128, ref.codes[w].shape).astype(F64)
        ref.scales[w] = F64(F32(0.02 * 2.0 ** r.uniform(-3, 1, ref.scales[w].shape)))
    return ref


def tables(r, lens, page):
    need = [-(-n // page) for n in lens]
    ids = r.permutation(sum(need) + 2)
    table = np.full((len(lens), max(max(need), 1)), -5, I32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, sum(need) + 2


def attention_wide(q, ref, table, start, lens):
    """-> (out, tolerance), all rows of a request and KV head as one matrix."""
    rows, heads, dim = q.shape
    kvh = ref.codes[0].shape[1]
    group = heads // kvh
    out, tol = np.full(q.shape, 7.0), np.zeros(q.shape)
    for b, total in enumerate(lens):
        n = start[b + 1] - start[b]
        if n == 0:
            continue
        t = np.arange(total)
        slots = table[b][t // ref.page] * ref.page + t % ref.page
        for g in range(kvh):
            k, v = (ref.values(w, slots)[:, g] for w in (0, 1))
            codes = np.abs(ref.codes[1][slots // ref.page, g, slots % ref.page]).cumsum(0)
            scale = ref.scales[1][slots // ref.page, g]
            for i0 in range(0, n, 256):
                i1 = min(i0 + 256, n)
                qq = q[start[b] + i0:start[b] + i1, g * group:(g + 1) * group].astype(F64).reshape(-1, dim)
                last = np.repeat(total - n + np.arange(i0, i1), group)
                seen = t[None, :] <= last[:, None]
                s = qq @ k.T / np.sqrt(dim)
                a = np.abs(qq) @ np.abs(k).T / np.sqrt(dim)
                top = np.where(seen, s, -np.inf).max(1, keepdims=True)
                e = np.where(seen, np.exp(np.minimum(s - top, 0)), 0.0)
                w = e / e.sum(1, keepdims=True)
                o = w @ v
                we = w * (2.0 ** -21 * a + 2.0 ** -22 * (np.abs(s) + np.abs(s - top)) + 2.0 ** -20)
                d = we @ np.abs(v) + we.sum(1, keepdims=True) * np.abs(o) + 2.0 ** -21 * (w @ np.abs(v))
                d += 2.0 ** -31 * (w * scale).max(1, keepdims=True) * codes[last]
                at = (slice(start[b] + i0, start[b] + i1), slice(g * group, (g + 1) * group))
                out[at], tol[at] = o.reshape(i1 - i0, group, dim), d.reshape(i1 - i0, group, dim)
    return out, tol


def compare(r, lens, fresh, heads, kvh, dim, page):
    table, pages = tables(r, lens, page)
    ref = random_cache(r, pages, kvh, page, dim)
    start = np.concatenate([[0], np.cumsum(fresh)]).astype(int)
    q = r.standard_normal((start[-1], heads, dim)).astype(F32)
    out = torch.full(q.shape, float("nan"), device="cuda")   # a row that nothing writes shows
    got = host(ops.attn_kv8_rows(dev(q), gpu_cache(ref), dev(table), dev(start, I32), dev(lens, I32), out=out))
    want, tol = attention_wide(q, ref, table, start, lens)
    ok = np.abs(got - want) <= tol
    assert np.all(ok), (np.argwhere(~ok)[0], int((~ok).any(axis=(1, 2)).sum()))


def row_tiles(fresh, heads, kvh):
    """Workgroups of the many-row kernel, before keys are cut."""
    g = heads // kvh
    return sum(-(-n * g // 128) for n in fresh if n * g > max(32, g)) * kvh


def test_more_row_tiles_than_the_card_takes():
    """Prompts whose keys are not cut (256 row tiles and more), a second, ragged one and single tokens beside them, whose
    pieces are joined four pairs to a wave."""
    r = np.random.default_rng(21)
    fresh, lens = [1, 2111, 1, 77, 2, 1], [700, 2111, 33, 400, 1500, 1]
    assert row_tiles(fresh, 16, 2) >= 256 and sum(fresh) * 16 > 16384
    compare(r, lens, fresh, 16, 2, 64, 64)


@pytest.mark.parametrize("heads,kvh,dim", [(16, 2, 64), (16, 2, 128), (24, 2, 256)])
def test_cut_prompts_joined_four_pairs_a_wave(heads, kvh, dim):
    """Few enough row tiles to be cut, and more than 16384 pairs with the single tokens beside them."""
    r = np.random.default_rng(dim)
    fresh = [1] * 120 + [500] + [1] * 110
    lens = list(r.integers(1, 400, 120)) + [900] + list(r.integers(200, 700, 110))
    if heads == 16:
        fresh[120], lens[120] = 860, 1300
    assert row_tiles(fresh, heads, kvh) <= 128 and sum(fresh) * heads > 16384
    compare(r, [int(n) for n in lens], fresh, heads, kvh, dim, 16)


@pytest.mark.parametrize("dim", [64, 128])
def test_cut_prompts_joined_a_pair_a_wave(dim):
    """2049 to 16384 pairs at the narrower heads; two prompts whose pieces differ in number."""
    r = np.random.default_rng(dim + 1)
    fresh, lens = [120, 1, 37, 9], [1200, 2500, 301, 40]
    assert 2048 < sum(fresh) * 16 <= 16384
    compare(r, lens, fresh, 16, 2, dim, 32)


@pytest.mark.parametrize("page", [8, 64])
def test_rows_of_no_request_are_left(page):
    """A part of a step's starts with all of its rows: the rows before the first request and behind the last stay as they
    are, whatever an earlier call has left in the workspace."""
    r = np.random.default_rng(page)
    heads, kvh, dim = 16, 2, 128
    lens, fresh = [1500, 900, 700], [40, 1, 3]
    table, pages = tables(r, lens, page)
    ref = random_cache(r, pages, kvh, page, dim)
    cache = gpu_cache(ref)
    start = np.concatenate([[0], np.cumsum(fresh)]).astype(int)
    q = r.standard_normal((start[-1] + 4, heads, dim)).astype(F32)
    ws = torch.zeros(ops.attn_kv8_workspace_bytes(len(q), 3, heads, kvh, dim), dtype=torch.uint8, device="cuda")
    out = torch.full(q.shape, 7.0, device="cuda")
    args = dict(workspace=ws, out=out)
    got = host(ops.attn_kv8_rows(dev(q), cache, dev(table), dev(start, I32), dev(lens, I32), **args))
    want, tol = attention_wide(q, ref, table, start, lens)
    assert np.all(np.abs(got - want) <= tol)
    for first in (1, 2, 3):   # the requests from `first` on, in a call of as many (the last ones idle)
        part = np.concatenate([start[first:], [start[-1]] * first])
        some = np.concatenate([table[first:], table[:first]])
        some_lens = lens[first:] + [0] * first
        out.fill_(7.0)
        got = host(ops.attn_kv8_rows(dev(q), cache, dev(some), dev(part, I32), dev(some_lens, I32), **args))
        want, tol = attention_wide(q, ref, some, part, some_lens)
        assert np.all(got[:part[0]] == 7.0) and np.all(got[part[-1]:] == 7.0)
        assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("up", [-20, 0, 10, 30])
@pytest.mark.parametrize("n", [2, 40])
def test_pages_of_zeros_keep_their_weight(n, up):
    """Pages whose values are all zero, of a whole tile and more, before and behind ones with values up to 2^up: what they
    take of the softmax stays, however small a value their scale (the smallest one) stands for."""
    r = np.random.default_rng(100 + n + up)
    page, heads, kvh, dim, zeros = 64, 8, 1, 64, 4
    total = page * (2 * zeros + 1)
    table, pages = tables(r, [total], page)
    ref = random_cache(r, pages, kvh, page, dim)
    for j in range(2 * zeros + 1):
        p = table[0, j]
        ref.scales[0][p] = F64(F32(7.0 / 800))
        if j == zeros:   # the page with values: scores some 7 (a factor of 2^10) above the others'
            ref.codes[0][p] = 100 + r.integers(-5, 6, ref.codes[0][p].shape)
            ref.scales[1][p] = 2.0 ** (up - 7)
        else:
            ref.codes[0][p] = r.integers(-5, 6, ref.codes[0][p].shape)
            ref.codes[1][p], ref.scales[1][p] = 0, kv8_ref.FLOOR
    q = (1 + 0.1 * r.standard_normal((n, heads, dim))).astype(F32)
    got = host(ops.attn_kv8_rows(dev(q), gpu_cache(ref), dev(table), dev([0, n], I32), dev([total], I32)))
    want, tol = attention_wide(q, ref, table, [0, n], [total])
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("fresh,lens", [([1, 3], [900, 40]), ([200, 1, 30], [200, 70, 1500]), ([1100], [1100])])
def test_output_in_the_place_of_the_gate(fresh, lens):
    """The same bits as apart, from one piece, several, and prompts cut and uncut."""
    r = np.random.default_rng(len(fresh))
    heads, kvh, dim, page = 16, 2, 128, 32
    table, pages = tables(r, lens, page)
    start = np.concatenate([[0], np.cumsum(fresh)]).astype(int)
    q, gate = (dev(r.standard_normal((start[-1], heads, dim)), F32) for _ in range(2))
    args = (q, gpu_cache(random_cache(r, pages, kvh, page, dim)), dev(table), dev(start, I32), dev(lens, I32))
    want = ops.attn_kv8_rows(*args, gate=gate)
    assert ops.attn_kv8_rows(*args, gate=gate, out=gate) is gate and torch.equal(gate, want)
