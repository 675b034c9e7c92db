"""Q/K norm and rotation by positions of several axes, against the formula in 64 bits.

Tolerance, from the roundings: x (r w) with r = rsqrt(mean + eps) carries the sum of squares (64 lanes' partial sums and six
levels: below 2^-21 of the sum, half of that of its root), the square root's 2 ulp and three products: 2^-20 of |x r w|. The
angle keeps 2^-25 of a revolution, 2 pi 2^-25 < 2^-22, and sine and cosine are within 2 ulp, 2^-22: a rotated pair is off by
(2^-20 + 2^-21 + 2^-22) of |a| + |b|, taken as 2^-19."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from qwen35_hip import _lib, ops

F32, I32 = np.float32, np.int32
gpu = pytest.mark.gpu


def dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).cuda()


def axes_of(sections, interleaved):
    if not interleaved:
        return np.repeat(np.arange(len(sections)), sections)
    left, out = list(sections), []
    while any(left):
        for a in range(len(sections)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return np.array(out)


def expected(x, w, pos, sections, interleaved, theta, eps):
    x = x.astype(np.float64)
    half = sum(sections)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    angle = pos.astype(np.float64)[axes_of(sections, interleaved)].T * theta ** (-np.arange(half) / half)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = y[..., :half].copy(), y[..., half:2 * half].copy()
    tol = 2.0 ** -20 * np.abs(y)
    tol[..., :half] = tol[..., half:2 * half] = 2.0 ** -19 * (np.abs(a) + np.abs(b))
    y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
    return y, tol


def run(r, rows, qh, kh, hd, sections, interleaved=True, theta=1e7, eps=1e-6, far=40000, shift=0):
    q, k = ((10.0 ** r.uniform(-2, 2, (rows, h, 1)) * r.standard_normal((rows, h, hd))).astype(F32) for h in (qh, kh))
    qw, kw = (r.uniform(-2, 2, hd).astype(F32) for _ in range(2))
    pos = r.integers(0, far, (len(sections), rows)).astype(I32)

    def moved(a):   # `shift` floats from a 16-byte boundary
        t = torch.empty(a.size + shift, device="cuda")
        t[shift:].copy_(dev(a).view(-1))
        return t[shift:].view(a.shape)
    tq, tk = moved(q), moved(k)
    ops.attn_qk_norm_mrope_rows(tq, tk, dev(qw), dev(kw), dev(pos), sections, interleaved=interleaved, theta=theta, eps=eps)
    torch.cuda.synchronize()
    for got, x, w in ((tq, q, qw), (tk, k, kw)):
        want, tol = expected(x, w, pos, sections, interleaved, float(F32(theta)), float(F32(eps)))
        assert np.all(np.abs(got.cpu().numpy() - want) <= tol + 1e-37)


@gpu
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("qh,kh,hd,sections", [
    (16, 2, 256, (11, 11, 10)), (24, 8, 128, (24, 20, 20)), (12, 12, 64, (16, 8, 8)), (3, 1, 256, (50, 40, 38)),
    (1, 1, 128, (4, 0, 0)), (5, 2, 64, (0, 3, 1)), (4, 4, 256, (32,)), (2, 1, 128, (8, 4, 2, 2)), (16, 2, 80, (8, 6, 6)),
    (2, 2, 96, (3, 3, 1)), (3, 1, 256, (5, 5, 5)), (1, 1, 2, (1,)), (2, 1, 512, (100, 20, 8)),
])
def test_layouts(qh, kh, hd, sections, interleaved):
    r = np.random.default_rng(hd + qh)
    for rows in (1, 2, 37):
        run(r, rows, qh, kh, hd, sections, interleaved)


@gpu
@pytest.mark.parametrize("far", [1, 2 ** 20, 2 ** 31 - 1])
def test_far_positions(far):
    """The angle's 2^-25 of a revolution holds while the 64-bit product does: past 2^31 / 2 pi revolutions 2^-25 is left too."""
    run(np.random.default_rng(far % 97), 65, 4, 2, 256, (11, 11, 10), far=far)
    run(np.random.default_rng(far % 89), 65, 4, 2, 128, (24, 20, 20), False, theta=1e4, far=far)


@gpu
def test_unaligned_and_many_rows():
    r = np.random.default_rng(0)
    run(r, 1000, 16, 2, 256, (11, 11, 10))
    run(r, 9, 3, 2, 256, (11, 11, 10), shift=1)
    run(r, 9, 3, 2, 64, (8, 8, 8), shift=3)


@gpu
def test_equal_axes_are_one_position():
    """A text token's axes agree: within fp32 angles of the form with one position."""
    r = np.random.default_rng(5)
    q, k = (dev(r.standard_normal((50, h, 256)).astype(F32)) for h in (16, 2))
    w = dev(r.uniform(0.5, 2, 256).astype(F32))
    pos = dev(np.arange(50) + 100, I32)
    q2, k2 = q.clone(), k.clone()
    ops.attn_qk_norm_mrope_rows(q, k, w, w, pos.expand(3, 50).contiguous(), (11, 11, 10))
    ops.attn_qk_norm_rope_rows(q2, k2, w, w, pos=pos)
    for a, b in ((q, q2), (k, k2)):   # an angle of up to 150 is off by 150 * 2^-24 = 2^-16.7, sizes are below 2 * 5
        assert float((a - b).abs().max()) <= 2.0 ** -16.7 * 20


@gpu
def test_queries_or_keys_alone_and_no_rows():
    r = np.random.default_rng(6)
    x, w = r.standard_normal((7, 4, 64)).astype(F32), r.uniform(0.5, 2, 64).astype(F32)
    pos = r.integers(0, 99, (3, 7)).astype(I32)
    want, tol = expected(x, w, pos, (8, 4, 4), True, 1e7, float(F32(1e-6)))
    none = torch.empty((7, 0, 64), device="cuda")
    for swap in (False, True):
        t = dev(x)
        ops.attn_qk_norm_mrope_rows(*((none, t) if swap else (t, none)), dev(w), dev(w), dev(pos), (8, 4, 4))
        torch.cuda.synchronize()
        assert np.all(np.abs(t.cpu().numpy() - want) <= tol)
    e = torch.empty((0, 4, 64), device="cuda")
    ops.attn_qk_norm_mrope_rows(e, e.clone(), dev(w), dev(w), torch.empty((3, 0), dtype=torch.int32, device="cuda"), (8, 4, 4))


@gpu
def test_non_finite_rows_stay_alone():
    r = np.random.default_rng(7)
    x = r.standard_normal((3, 6, 256)).astype(F32)
    x[1, 2, 200] = np.nan
    w = np.ones(256, F32)
    t, k = dev(x), dev(x[:, :2])
    ops.attn_qk_norm_mrope_rows(t, k, dev(w), dev(w), dev(np.zeros((3, 3)), I32), (11, 11, 10))
    torch.cuda.synchronize()
    bad = np.isnan(t.cpu().numpy())
    assert bad[1, 2].all() and bad.sum() == 256 and not np.isnan(k.cpu().numpy()).any()


@gpu
def test_wrong_tensors_are_refused():
    z = lambda *s: torch.zeros(s, device="cuda")
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    ok = dict(q=z(3, 4, 64), k=z(3, 2, 64), q_weight=z(64), k_weight=z(64), pos=i(3, 3), sections=(8, 4, 4))
    for bad in (dict(pos=i(2, 3)), dict(pos=i(3, 4)), dict(pos=z(3, 3)), dict(k=z(2, 2, 64)), dict(q_weight=z(63)),
                dict(q=z(3, 4, 128)[:, :, :64])):
        with pytest.raises(ValueError):
            ops.attn_qk_norm_mrope_rows(**{**ok, **bad})
    for bad in (dict(sections=(0, 0, 0)), dict(sections=(30, 2, 1)), dict(sections=(8, -4, 4)), dict(theta=0.0)):
        with pytest.raises(_lib.QwenError):
            ops.attn_qk_norm_mrope_rows(**{**ok, **bad})
    with pytest.raises(_lib.QwenError, match="overlap"):
        x = z(3, 6, 64)
        ops.attn_qk_norm_mrope_rows(x.view(-1)[:768].view(3, 4, 64), x.view(-1)[640:1024].view(3, 2, 64), z(64), z(64), i(3, 3),
                                    (8, 4, 4))
