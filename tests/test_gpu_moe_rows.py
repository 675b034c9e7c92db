"""The routed experts of many tokens: pairs grouped by expert (compared exactly), the experts' products (against 64 bits).

The tolerance of a product follows its roundings. With B = sum_k (|d sc q| + |dmin m|) |x_k| over a row: the two fp16
parts of x lose 2^-22 of each term, and the fp32 sums, some 18 roundings a block of partial sums that random signs keep
below B / 36 over 8 blocks (B / 9 over 2), as much again: 2^-21 B. SwiGLU adds its own 2^-18 (silu's documented 2.8e-6),
and passes the products' errors on with |silu'| <= 1.1."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from qwen35_hip import _lib, ops, synth

pytestmark = pytest.mark.gpu
F32, F64, I32 = np.float32, np.float64, np.int32


def dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).cuda()


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


# ------------------------------------------------------------------ grouping
@pytest.mark.parametrize("pairs,experts", [(0, 4), (1, 1), (8, 256), (63, 3), (64, 64), (65, 1), (1000, 256), (1024, 1024),
                                           (1025, 60), (4097, 7), (32768, 256), (20000, 1000)])
def test_group(pairs, experts):
    r = np.random.default_rng(pairs + experts)
    idx = (r.integers(0, experts, pairs) * r.integers(0, 2, pairs)).astype(I32)   # expert 0 has half of them
    order, starts = (host(t) for t in ops.moe_group_rows(dev(idx), experts))
    assert np.array_equal(order, np.argsort(idx, kind="stable"))
    assert np.array_equal(starts, np.concatenate([[0], np.cumsum(np.bincount(idx, minlength=experts))]))


def test_group_ids_outside():
    r = np.random.default_rng(0)
    idx = r.integers(-2, 12, 3000).astype(I32)
    idx[::97], idx[5::101] = 2 ** 31 - 1, -2 ** 31
    order, starts = (host(t) for t in ops.moe_group_rows(dev(idx), 10))
    key = np.where((idx >= 0) & (idx < 10), idx, 10)
    assert np.array_equal(order, np.argsort(key, kind="stable"))
    assert np.array_equal(starts, np.concatenate([[0], np.cumsum(np.bincount(key, minlength=11)[:10])]))


# ------------------------------------------------------------------ the products
def table(kind, rows, cols, seed):
    return (synth.q4k_table if kind == "Q4_K" else synth.q6k_table)(rows, cols, seed_tensor=seed)


def decode(kind, raw, rows, cols):
    """Values and the sizes of their terms, in 64 bits."""
    if kind == "Q4_K":
        b = raw.reshape(-1, 144).astype(np.int64)
        half = raw.reshape(-1, 144)[:, :4].copy().view(np.float16).astype(F64)
        i = np.arange(256)
        g = i // 32
        sc = np.where(g < 4, b[:, 4 + g % 4] & 63, (b[:, 12 + g % 4] & 15) | ((b[:, 4 + g % 4] >> 6) << 4))
        mn = np.where(g < 4, b[:, 8 + g % 4] & 63, (b[:, 12 + g % 4] >> 4) | ((b[:, 8 + g % 4] >> 6) << 4))
        q = (b[:, 16 + 32 * (i // 64) + i % 32] >> (4 * (g % 2))) & 15
        p, m = half[:, :1] * sc * q, half[:, 1:] * mn
        return (p - m).reshape(rows, cols), (np.abs(p) + np.abs(m)).reshape(rows, cols)
    b = raw.reshape(-1, 210).astype(np.int64)
    d = raw.reshape(-1, 210)[:, 208:].copy().view(np.float16).astype(F64)
    i = np.arange(256)
    h, quarter, c = i // 128, i % 128 // 32, i % 32
    q = ((b[:, 64 * h + 32 * (quarter % 2) + c] >> (4 * (quarter // 2))) & 15) | (
        ((b[:, 128 + 32 * h + c] >> (2 * quarter)) & 3) << 4)
    sc = b[:, 192 + i // 16]
    w = d * np.where(sc > 127, sc - 256, sc) * (q - 32)
    return w.reshape(rows, cols), np.abs(w).reshape(rows, cols)


def silu(g):
    return g / (1.0 + np.exp(-g))


class Layer:
    def __init__(self, experts, inter, width, kind, down, seed=3):
        self.e, self.inter, self.width, self.kind, self.down = experts, inter, width, kind, down
        self.raw = [table(kind, experts * inter, width, seed), table(kind, experts * inter, width, seed + 8),
                    table(down, experts * width, inter, seed + 16)]
        dims = [(kind, inter, width), (kind, inter, width), (down, width, inter)]
        self.w = [decode(k, raw, experts * m, c) for raw, (k, m, c) in zip(self.raw, dims)]
        self.dev = [dev(raw) for raw in self.raw]

    def expert(self, which, e):
        rows = self.width if which == 2 else self.inter
        return tuple(a[e * rows:(e + 1) * rows] for a in self.w[which])

    def call(self, idx, weights, x, **kw):
        order, starts = ops.moe_group_rows(dev(idx), self.e)
        return ops.moe_experts_rows(self.dev[0], self.dev[1], self.kind, self.dev[2], self.down, self.e, order, starts,
                                    dev(weights), dev(x), self.inter, **kw)

    def reference(self, idx, weights, x):
        out, tol = np.zeros(x.shape, F64), np.zeros(x.shape, F64)
        x = x.astype(F64)
        for e in range(self.e):
            t, j = np.nonzero(idx == e)
            if len(t) == 0:
                continue
            (wg, ag), (wu, au), (wd, ad) = (self.expert(i, e) for i in range(3))
            xs = x[t]
            g, u = xs @ wg.T, xs @ wu.T
            dg, du = 2.0 ** -21 * (np.abs(xs) @ ag.T), 2.0 ** -21 * (np.abs(xs) @ au.T)
            h = silu(g) * u
            dh = 1.1 * dg * np.abs(u) + np.abs(silu(g)) * du + 1.1 * dg * du + 2.0 ** -18 * np.abs(h)
            y = h @ wd.T
            dy = dh @ np.abs(wd).T + 2.0 ** -21 * (np.abs(h) @ ad.T)
            a = weights[t, j].astype(F64)[:, None]
            np.add.at(out, t, a * y)
            np.add.at(tol, t, np.abs(a) * (dy + 2.0 ** -22 * np.abs(y)))
        return out, tol


def routing(r, rows, top, experts, sizes=None):
    """Ids (of a token all different, as a top-k gives them) and weights; sizes: pairs of the first experts, the rest
    spread over the others."""
    if sizes is not None:
        idx = np.repeat(np.arange(len(sizes)), sizes).astype(I32).reshape(rows, top)
    else:
        idx = np.stack([r.permutation(experts)[:top] for _ in range(rows)]).astype(I32)
    w = r.uniform(0.05, 1, (rows, top)).astype(F32)
    return idx, w / w.sum(1, keepdims=True)


def check(layer, idx, w, x, **kw):
    got = host(layer.call(idx, w, x, **kw))
    want, tol = layer.reference(idx, w, x)
    err = np.abs(got - want)
    assert np.all(err <= tol), (float((err / np.maximum(tol, 1e-300)).max()), np.argwhere(~(err <= tol))[0])
    # and as an fp32 result should be, against the rows' size
    rms = np.sqrt((want ** 2).mean(1, keepdims=True))
    assert np.all(err <= 1e-5 * np.maximum(rms, 1e-30)), float((err / np.maximum(rms, 1e-30)).max())
    return got


@pytest.mark.parametrize("kind,down", [("Q4_K", "Q4_K"), ("Q6_K", "Q6_K"), ("Q4_K", "Q6_K")])
@pytest.mark.parametrize("rows,top,experts,inter,width", [
    (1, 1, 1, 256, 256), (1, 8, 16, 512, 2048), (5, 8, 16, 512, 2048), (3, 2, 7, 256, 768),       # groups of a few pairs
    (2, 3, 40, 1280, 512), (4, 4, 9, 2048, 1024), (3, 2, 4, 256, 2304), (9, 3, 5, 2560, 256),      # and rows past 8 blocks
    (40, 4, 16, 256, 512), (33, 3, 5, 512, 256), (21, 8, 12, 1280, 512),                           # of 10 to 20
    (100, 4, 6, 512, 2048), (130, 1, 2, 256, 256), (67, 2, 3, 768, 768),                           # of 45 and more
])
def test_experts(kind, down, rows, top, experts, inter, width):
    r = np.random.default_rng(rows + inter)
    idx, w = routing(r, rows, top, experts)
    check(Layer(experts, inter, width, kind, down), idx, w, (0.05 * r.standard_normal((rows, width))).astype(F32))


@pytest.mark.parametrize("kind", ["Q4_K", "Q6_K"])
@pytest.mark.parametrize("sizes", [
    [0, 1, 15, 16, 17, 0, 2, 1, 4, 0, 3, 5], [31, 32, 33, 1, 0, 7, 8, 16], [63, 64, 65, 0, 1, 127], [129, 191, 0, 0],
    [0, 0, 200], [300, 0, 1, 1, 1, 1, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0]])
def test_experts_ragged(kind, sizes):
    """Groups at the edges of every tile, empty ones, and one that holds all."""
    r = np.random.default_rng(sum(sizes))
    rows = sum(sizes)
    idx, w = routing(r, rows, 1, len(sizes), sizes)
    check(Layer(len(sizes), 256, 512, kind, kind), idx, w, (0.05 * r.standard_normal((rows, 512))).astype(F32))


@pytest.mark.parametrize("kind", ["Q4_K", "Q6_K"])
def test_experts_tiles_of_every_size(kind):
    """Groups around each number of sixteens that a tile can have, and the even tiles of larger ones; odd numbers of blocks."""
    sizes = [24, 47, 48, 49, 63, 79, 80, 81, 96, 97, 112, 145]
    r = np.random.default_rng(99)
    rows = sum(sizes)
    idx, w = routing(r, rows, 1, len(sizes), sizes)
    check(Layer(len(sizes), 256, 768, kind, kind), idx, w, (0.05 * r.standard_normal((rows, 768))).astype(F32))


def test_experts_rows_of_many_sizes():
    """Rows of x from 1e-30 to 1e10, one of zeros, one whose elements span 2^40."""
    r = np.random.default_rng(7)
    rows = 12
    x = r.standard_normal((rows, 512)) * 10.0 ** np.linspace(-30, 3, rows)[:, None]
    x[4] = 0
    x[5] = r.standard_normal(512) * 2.0 ** r.uniform(-40, 0, 512)
    idx, w = routing(r, rows, 3, 6)
    layer = Layer(6, 256, 512, "Q4_K", "Q4_K")
    got = host(layer.call(idx, w, x.astype(F32)))
    want, tol = layer.reference(idx, w, x.astype(F32))
    assert np.all(got[4] == 0)
    # the parts' absolute step, 2^-39 of a row's largest element, over 512 products (row 5; others are far above it)
    big = max(np.abs(layer.w[i][0]).max() for i in range(2))
    assert np.all(np.abs(got - want) <= tol + 1e-37 + 2.0 ** -39 * 512 * big * np.abs(x).max(1, keepdims=True) *
                  np.abs(layer.w[2][0]).max() * 256)


@pytest.mark.parametrize("rows", [3, 40, 150])
def test_experts_non_finite_rows(rows):
    """An infinity follows its products and sums into the outputs of its own row; a NaN fills its row."""
    r = np.random.default_rng(rows)
    x = (0.05 * r.standard_normal((rows, 256))).astype(F32)
    x[1, 7], x[2, 9] = np.inf, np.nan
    idx, w = routing(r, rows, 1, 3)
    layer = Layer(3, 256, 256, "Q4_K", "Q6_K")
    got = host(layer.call(idx, w, x))
    assert np.all(np.isnan(got[2]))
    rest = np.array([t for t in range(rows) if t not in (1, 2)])
    want, tol = layer.reference(idx[rest], w[rest], x[rest])
    assert np.all(np.abs(got[rest] - want) <= tol)
    with np.errstate(all="ignore"):
        (wg, _), (wu, _), (wd, _) = (layer.expert(i, idx[1, 0]) for i in range(3))
        xs = x[1].astype(F64)
        g, u = (wg * xs).sum(1), (wu * xs).sum(1)
        y = (wd * (silu(g) * u)).sum(1)
    assert np.array_equal(np.isnan(got[1]), np.isnan(y)) and np.array_equal(np.isinf(got[1]), np.isinf(y))


@pytest.mark.parametrize("rows,top", [(4, 3), (200, 2)])
def test_experts_ids_outside(rows, top):
    """A token with an id outside the experts has a NaN row (its weight may be finite), the others their values."""
    r = np.random.default_rng(rows)
    idx, w = routing(r, rows, top, 5)
    bad = idx.copy()
    bad[1, 0], bad[rows - 1, top - 1] = -1, 5
    x = (0.05 * r.standard_normal((rows, 256))).astype(F32)
    layer = Layer(5, 256, 256, "Q4_K", "Q4_K")
    ws = torch.full((ops.moe_experts_rows_workspace_bytes(rows, top, 5, 256, 256),), 0x7f, dtype=torch.uint8, device="cuda")
    got = host(layer.call(bad, w, x, workspace=ws))
    want, tol = layer.reference(bad, w, x)
    ok = np.ones(rows, bool)
    ok[[1, rows - 1]] = False
    assert np.all(np.isnan(got[~ok])) and np.all(np.abs(got - want)[ok] <= tol[ok])
    allbad = host(layer.call(np.full_like(idx, -1), w, x, workspace=ws))
    assert np.all(np.isnan(allbad))


def test_experts_equal_the_decode_step():
    """The same tokens one at a time through the decode entry points: equal within both sides' roundings."""
    r = np.random.default_rng(1)
    layer = Layer(16, 512, 2048, "Q4_K", "Q4_K")
    idx, w = routing(r, 6, 8, 16)
    x = (0.05 * r.standard_normal((6, 2048))).astype(F32)
    got = check(layer, idx, w, x)
    for t in range(6):
        h, _ = ops.moe_expert_swiglu(layer.dev[0], layer.dev[1], "Q4_K", 16 * 512 * 2048, 512 * 2048, 16, dev(idx[t]),
                                     dev(x[t]), 512, 2048)
        y = ops.moe_expert_matmul(layer.dev[2], "Q4_K", 16 * 512 * 2048, 512 * 2048, 16, dev(idx[t]), h, 512, 2048, 512)
        out = torch.zeros((1, 2048), device="cuda")
        ops.moe_weighted_sum_rows(out, y.view(1, 8, 2048), dev(w[t]).view(1, 8))
        _, tol = layer.reference(idx[t:t + 1], w[t:t + 1], x[t:t + 1])
        assert np.all(np.abs(host(out) - got[t]) <= 2 * tol)


def test_experts_in_a_graph_and_on_a_stream():
    """Captured once, replayed with other routings and rows: each replay the eager call's bits, and no other bits on
    another stream; nothing is kept in the workspace."""
    r = np.random.default_rng(2)
    layer = Layer(9, 256, 512, "Q6_K", "Q4_K")
    rows, top = 70, 3
    idx, w = dev(np.zeros((rows, top)), I32), dev(np.zeros((rows, top)), F32)
    x, out = torch.zeros((rows, 512), device="cuda"), torch.zeros((rows, 512), device="cuda")
    order, starts = torch.zeros(rows * top, dtype=torch.int32, device="cuda"), torch.zeros(10, dtype=torch.int32, device="cuda")
    ws = torch.zeros(ops.moe_experts_rows_workspace_bytes(rows, top, 9, 512, 256), dtype=torch.uint8, device="cuda")

    def step(out):
        ops.moe_group_rows(idx, 9, order=order, starts=starts)
        return ops.moe_experts_rows(layer.dev[0], layer.dev[1], "Q6_K", layer.dev[2], "Q4_K", 9, order, starts, w, x, 256,
                                    out=out, workspace=ws)

    step(out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(out)
    for i in range(4):
        hi, hw = routing(r, rows, top, 9)
        hx = (0.05 * r.standard_normal((rows, 512))).astype(F32)
        idx.copy_(dev(hi)), w.copy_(dev(hw)), x.copy_(dev(hx))
        ws.fill_(255)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step(torch.empty_like(out)))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            again = step(torch.empty_like(out))
        s.synchronize()
        assert torch.equal(got, again)
        want, tol = layer.reference(hi, hw, hx)
        assert np.all(np.abs(host(got) - want) <= tol)


def test_refusals():
    layer = Layer(2, 256, 256, "Q4_K", "Q4_K")
    i, f = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.ones((1, 1), device="cuda")
    x = torch.zeros((1, 256), device="cuda")
    order, starts = ops.moe_group_rows(i, 2)
    call = lambda **kw: ops.moe_experts_rows(**{**dict(
        w_gate=layer.dev[0], w_up=layer.dev[1], ggml_type="Q4_K", w_down=layer.dev[2], down_type="Q4_K", n_experts=2,
        order=order, starts=starts, weights=f, x=x, inter=256), **kw})
    call()
    with pytest.raises(ValueError):
        call(ggml_type="Q6_K")      # the tensor is too small for it
    with pytest.raises(ValueError):
        call(starts=starts[:2].clone())
    with pytest.raises(ValueError):
        call(x=torch.zeros((2, 256), device="cuda"))
    with pytest.raises(_lib.QwenError, match="workspace"):
        call(workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))
    with pytest.raises(_lib.QwenError, match="out is x"):
        call(out=x)
    with pytest.raises(_lib.QwenError, match="experts"):
        ops.moe_group_rows(i, 1025)
    assert call(weights=f[:0], x=x[:0], order=order[:0]).shape == (0, 256)
