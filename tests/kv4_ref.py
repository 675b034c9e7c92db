"""Plain 64-bit forms of the paged 4-bit cache and of the attention over it, on the host, from their definitions."""

from __future__ import annotations

import numpy as np

F64, F32 = np.float64, np.float32
FLOOR = 2.0 ** -100


def bf16_bits(x):
    """Bits of float32 numbers that are bf16 ones."""
    b = np.asarray(x, F32).view(np.uint32)
    assert not np.any((b & 0xffff) & np.where(np.isnan(x), 0, 0xffff))
    return (b >> 16).astype(np.uint16)


def bf16_down(x):
    """The largest bf16 that is at most x (float32)."""
    b = np.asarray(x, F32).view(np.uint32)
    cut = b & np.uint32(0xffff0000)
    return np.where((b >> 31 == 1) & (cut != b), cut + np.uint32(0x10000), cut).astype(np.uint32).view(F32)


def bf16_up(x):
    """The smallest bf16 that is at least x (float64, positive)."""
    b = np.asarray(x, F64).astype(F32).view(np.uint32)
    up = (((b.astype(np.uint64) + 0xffff) >> 16) << 16).astype(np.uint32)
    return np.where(up.view(F32).astype(F64) < x, up + np.uint32(0x10000), up).astype(np.uint32).view(F32)


def quantize(x):
    """x [..., n] -> codes, scale, min (float64) of the groups of n; a group that is not finite has scale NaN."""
    x = np.asarray(x, F32)
    with np.errstate(all="ignore"):
        low = bf16_down(x.min(-1))
        ok = np.all(np.isfinite(x), axis=-1) & np.isfinite(low)
        low = np.where(ok, low, 0).astype(F32) + F32(0)   # a zero is +0
        clean = np.where(ok[..., None], x, 0).astype(F64)
        step = np.maximum((clean.max(-1) - low.astype(F64)) / 15.0, FLOOR)
        scale = bf16_up(step).astype(F64)
        codes = np.clip(np.rint((clean - low.astype(F64)[..., None]) / scale[..., None]), 0, 15)
    return np.where(ok[..., None], codes, 0), np.where(ok, scale, np.nan), low.astype(F64)


class Cache:
    """codes [pages, heads, page, dim], scale and min [pages, heads, page, groups] of keys (groups of 64) and values (one)."""

    def __init__(self, pages, heads, page, dim):
        self.page, self.pages, self.dim = page, pages, dim
        self.codes = [np.zeros((pages, heads, page, dim)) for _ in range(2)]
        self.scale = [np.zeros((pages, heads, page, g)) for g in (dim // 64, 1)]
        self.low = [np.zeros((pages, heads, page, g)) for g in (dim // 64, 1)]

    def store(self, which, x, slots):
        groups = self.scale[which].shape[-1]
        for i, s in enumerate(np.asarray(slots).tolist()):
            if 0 <= s < self.pages * self.page:
                p, o = divmod(s, self.page)
                c, sc, low = quantize(np.asarray(x[i], F32).reshape(x.shape[1], groups, -1))
                self.codes[which][p, :, o] = c.reshape(x.shape[1], -1)
                self.scale[which][p, :, o], self.low[which][p, :, o] = sc, low

    def values(self, which, slots):
        """[rows, heads, dim] in 64 bits."""
        s = np.asarray(slots)
        p, o = s // self.page, s % self.page
        n = self.dim // self.scale[which].shape[-1]
        wide = [np.repeat(t[which][p, :, o], n, axis=-1) for t in (self.scale, self.low)]
        return wide[1] + wide[0] * self.codes[which][p, :, o]

    def arrays(self):
        """k, v, k_scale, k_min, v_scale, v_min as the library lays them out (bf16 as bits)."""
        pages, heads, page, dim = self.codes[0].shape
        ng = dim // 64

        def words(c):   # [..., 8] codes -> uint32: elements 0, 2, 4, 6, 1, 3, 5, 7 in nibbles 0..7
            out = np.zeros(c.shape[:-1], np.uint32)
            for n, j in enumerate((0, 2, 4, 6, 1, 3, 5, 7)):
                out |= c[..., j].astype(np.uint32) << np.uint32(4 * n)
            return out
        k = words(self.codes[0].reshape(pages, heads, page, ng, 4, 2, 8)).transpose(0, 1, 2, 4, 3, 5)   # [.., lk, g, h]
        v = words(self.codes[1].reshape(pages, heads, page // 8, 8, dim).swapaxes(-1, -2))
        ks = self.scale[0].reshape(pages, heads, page // 8, 8, ng).swapaxes(-1, -2)
        return (np.ascontiguousarray(k).view(np.uint8).reshape(pages, heads, page, dim // 2),
                np.ascontiguousarray(v).view(np.uint8).reshape(pages, heads, page // 8, dim, 4), bf16_bits(ks),
                bf16_bits(self.low[0]), bf16_bits(self.scale[1][..., 0]), bf16_bits(self.low[1][..., 0]))


def attention(q, cache, table, row_start, kv_len, gate=None):
    """-> (out, tolerance) [rows, heads, dim]; rows of no request hold 7.

    The tolerance counts the roundings of an fp32 evaluation whose products carry 22 bits over the parts that a value is
    made of, scale * code and min, whose magnitudes A = |scale| code + |min| stand for |value|. A score s = q.k / sqrt(D):
    2^-21 sum |q| A / sqrt(D) for the products, their sums and the scaling, and as an fp32 number that is rounded when it is
    scaled and when the reference is subtracted 2^-22 (|s| + |s - max|); its exponential by that and 2^-20. An output: those,
    weighted with |v - out|, and 2^-21 of sum p A (second product, its sums, the division). Of a weight p scale, its two fp16
    parts keep 22 bits: 2^-22 of it, times |code - 8| <= 8 as codes are summed, where the rest of a value, p (min + 8 scale), is
    an fp32 number that does not share that error: 2^-19 of sum p scale, which A does not cover where min and code are small.
    A weight p scale, as two fp16 parts, also has an absolute step, half the spacing of fp16's smallest numbers, 2^-25: times
    2^-6 in units of a reference that the largest p max(|min|, 16 scale, 2^-40) is at least half of. That is 2^-30 of the
    largest w max(..) with the normalised weights w, met by the codes."""
    rows, heads, dim = q.shape
    kvh = cache.codes[0].shape[1]
    out, tol = np.full(q.shape, 7.0), np.zeros(q.shape)
    for b in range(len(kv_len)):
        n, total = row_start[b + 1] - row_start[b], kv_len[b]
        t = np.arange(total)
        slots = np.asarray(table[b])[t // cache.page] * cache.page + t % cache.page if total else t
        p, o = slots // cache.page, slots % cache.page
        parts = []
        for w in (0, 1):
            rep = dim // cache.scale[w].shape[-1]
            c = cache.codes[w][p, :, o] if total else np.zeros((0, kvh, dim))
            sc, low = ((np.repeat(x[w][p, :, o], rep, axis=-1) if total else c) for x in (cache.scale, cache.low))
            parts.append((low + sc * c, sc * c + np.abs(low), c, np.maximum(np.maximum(16 * sc, np.abs(low)), 2.0 ** -40), sc))
        (k, ka, _, _, _), (v, va, vc, vm, vs) = parts
        for i in range(n):
            row, pos = row_start[b] + i, total - n + i
            for h in range(heads):
                if pos < 0:
                    out[row, h] = 0.0
                    continue
                g = h // (heads // kvh)
                sl = np.s_[:pos + 1, g]
                qq = q[row, h].astype(F64)
                s = k[sl] @ qq / np.sqrt(dim)
                a = ka[sl] @ np.abs(qq) / np.sqrt(dim)
                e = np.exp(s - s.max())
                w = e / e.sum()
                y = w @ v[sl]
                eps = 2.0 ** -21 * a + 2.0 ** -22 * (np.abs(s) + np.abs(s - s.max())) + 2.0 ** -20
                out[row, h] = y
                tol[row, h] = (w * eps) @ np.abs(v[sl] - y) + 2.0 ** -21 * (w @ va[sl])
                tol[row, h] += 2.0 ** -19 * (w @ vs[sl])
                tol[row, h] += 2.0 ** -30 * (w * vm[sl][:, 0]).max() * vc[sl].sum(axis=0)
    if gate is not None:
        live = row_start[len(kv_len)]
        sg = 1.0 / (1.0 + np.exp(-gate[:live].astype(F64)))
        # the sigmoid's own error, 2^-24 |gate| + 3 ulp, of the product
        tol[:live] = tol[:live] * sg + np.abs(out[:live]) * sg * (2.0 ** -24 * np.abs(gate[:live]) + 2.0 ** -21)
        out[:live] *= sg
    return out, tol
