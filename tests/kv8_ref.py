"""Plain 64-bit forms of the paged 8-bit cache operators, on the host: page bookkeeping, quantization, attention."""

from __future__ import annotations

import numpy as np

F64, F32, I8 = np.float64, np.float32, np.int8
FLOOR = 2.0 ** -100


def plan(cached, fresh, table, free, head, page, rows):
    table = np.array(table, dtype=np.int64).copy()
    start, lens, slots, pos, head0, used, short = [0], [], [], [], head, head, False
    at = max(0, min(head, len(free)))
    for b, (c, n) in enumerate(zip(cached, fresh)):
        c, n = max(int(c), 0), max(int(n), 0)
        have = -(-c // page)
        room = c + n <= page * table.shape[1] and start[-1] + n <= rows
        need = -(-(c + n) // page) - have if n and room else 0
        if need and (short or at + need > len(free)):
            short, granted = True, False
        else:
            granted = room
        if granted and need:
            table[b, have:have + need] = free[at:at + need]
            at += need
            used = at
        lens.append(c + n if granted else 0)
        start.append(start[-1] + n)
        for t in range(c, c + min(n, rows)):
            pos.append(t)
            slots.append(int(table[b, t // page]) * page + t % page if granted else -1)
    start = [min(s, 2 ** 31 - 1) for s in start]
    slots, pos = slots[:rows] + [-1] * (rows - len(slots)), pos[:rows] + [0] * (rows - len(pos))
    return table, start, lens, slots, pos, used if used != head0 else head0


class Cache:
    """codes [pages, heads, page, dim] of keys and values, scales [pages, heads]; values in token order."""

    def __init__(self, pages, heads, page, dim):
        self.page = page
        self.codes = [np.zeros((pages, heads, page, dim), F64) for _ in range(2)]
        self.scales = [np.zeros((pages, heads), F64) for _ in range(2)]

    def store(self, which, x, slots):
        codes, scales, P = self.codes[which], self.scales[which], self.page
        x = x.astype(F64)
        i, total = 0, codes.shape[0] * P
        while i < len(slots):
            s = int(slots[i])
            if s < 0 or s >= total:
                i += 1
                continue
            j = i + 1
            while j < len(slots) and slots[j] == slots[j - 1] + 1 and slots[j] // P == s // P:
                j += 1
            p, o = divmod(s, P)
            for h in range(codes.shape[1]):
                run = x[i:j, h]
                old = scales[p, h] if o else 0.0
                if not np.all(np.isfinite(run)) or np.isnan(old):
                    scales[p, h] = np.nan
                    codes[p, h, o:o + j - i] = 0
                    continue
                top = F64(F32(np.abs(run).max() / 127.0))
                new = max(old, top, FLOOR)
                codes[p, h, :o] = np.rint(codes[p, h, :o] * F64(F32(old / new)))
                codes[p, h, o:o + j - i] = np.clip(np.rint(run / new), -127, 127)
                scales[p, h] = new
            i = j

    def values(self, which, slots):
        """[rows, heads, dim] in 64 bits."""
        s = np.asarray(slots)
        p, o = s // self.page, s % self.page
        return self.codes[which][p, :, o] * self.scales[which][p][:, :, None]


def attention(q, cache, table, row_start, kv_len, gate=None):
    """-> (out, tolerance) [rows, heads, dim]. The tolerance follows the roundings of an fp32 evaluation whose products
    carry 22 bits: a score s with sum A of |q k| / sqrt(D) is off by up to 2^-21 A and, as an fp32 number that is
    rounded when it is scaled and when the reference is subtracted, by 2^-22 |s| + 2^-22 |s - max|; its exponential by
    that and 2^-20; an output by those, weighted with |v - out|, and by 2^-21 of
    sum p |v| (the second product and the division).
    A weight also has an absolute step. With p_t v_scale_t, relative to a reference that keeps the largest of them
    between 1 and 2^8, times 2^6 as two fp16 parts, what the parts lose is at most half the spacing of fp16's smallest
    numbers, 2^-25, that is 2^-31 of that reference. It meets the codes: sum_t 2^-31 |code_t| over the same sum
    l of p_t, and 1 / l <= max_t (p_t v_scale_t) / l = max_t (w_t v_scale_t) with the normalised weights w."""
    rows, heads, dim = q.shape
    kvh = cache.codes[0].shape[1]
    out, tol = np.full(q.shape, 7.0), np.zeros(q.shape)
    for b in range(len(kv_len)):
        n, total = row_start[b + 1] - row_start[b], kv_len[b]
        t = np.arange(total)
        slots = np.asarray(table[b])[t // cache.page] * cache.page + t % cache.page if total else t
        k, v = (cache.values(w, slots) for w in (0, 1)) if total else (np.zeros((0, kvh, dim)),) * 2
        codes = np.abs(cache.codes[1][slots // cache.page, :, slots % cache.page]) if total else k
        scale = cache.scales[1][slots // cache.page] if total else k
        for i in range(n):
            row, p = row_start[b] + i, total - n + i
            for h in range(heads):
                if p < 0:
                    out[row, h] = 0.0
                    continue
                g = h // (heads // kvh)
                kk, vv, qq = k[:p + 1, g], v[:p + 1, g], q[row, h].astype(F64)
                s = kk @ qq / np.sqrt(dim)
                a = np.abs(kk) @ np.abs(qq) / np.sqrt(dim)
                e = np.exp(s - s.max())
                w = e / e.sum()
                o = w @ vv
                eps = 2.0 ** -21 * a + 2.0 ** -22 * (np.abs(s) + np.abs(s - s.max())) + 2.0 ** -20
                out[row, h] = o
                tol[row, h] = (w * eps) @ np.abs(vv - o) + 2.0 ** -21 * (w @ np.abs(vv))
                tol[row, h] += 2.0 ** -31 * (w * scale[:p + 1, g]).max() * codes[:p + 1, g].sum(axis=0)
    if gate is not None:
        live = row_start[len(kv_len)]
        sg = 1.0 / (1.0 + np.exp(-gate[:live].astype(F64)))
        # the sigmoid's own error, 2^-24 |gate| + 3 ulp, of the product
        tol[:live] = tol[:live] * sg + np.abs(out[:live]) * sg * (2.0 ** -24 * np.abs(gate[:live]) + 2.0 ** -21)
        out[:live] *= sg
    return out, tol
