"""The routed experts with small groups, at sizes where a workgroup goes through many row tiles and over the borders of
several experts: every buffer of weights in flight is used again, the sums' two buffers many times, and workgroups end at
different turns. (256 workgroups share all tiles' turns; fewer than some 40 tiles give each of them two or three.)

Weights are made and decoded on the GPU, the reference is in 64 bits there. Tolerances: with B = sum_k (|d sc q| + |dmin m|)
|x_k| a product is off by 2^-21 B (2^-22 from the two fp16 parts of x, as much from the fp32 sums), SwiGLU by 2^-18 of its
value, and it passes the products' errors on with |silu'| <= 1.1; a weighted sum of k products rounds each by 2^-22."""

from __future__ import annotations

import pytest
import torch

from qwen35_hip import ops

pytestmark = pytest.mark.gpu
F64, I32, U8 = torch.float64, torch.int32, torch.uint8
BLOCK = {"Q4_K": 144, "Q6_K": 210}


def weights(g, kind, n):
    """n elements with scales and codes of every value, around zero and of a size of about 0.02."""
    nb = n // 256
    b = torch.randint(0, 256, (nb, BLOCK[kind]), generator=g, device="cuda", dtype=U8)
    d = 0.7 + 0.6 * torch.rand((nb, 2), generator=g, device="cuda")
    if kind == "Q4_K":   # (d sc) q - dmin m, sc and m up to 63, q up to 15: the same size where dmin is 7.5 d
        b[:, :4] = (d * torch.tensor([1.0, 7.5], device="cuda") * (0.02 / 209)).half().view(U8)
    else:                # (d sc) (q - 32), sc from -128 to 127
        b[:, 208:] = (d[:, :1] * (0.02 / 1500)).half().view(U8)
    return b.view(-1)


def decode(raw, kind, rows, cols):
    """Values and the sizes of their terms."""
    raw = raw.view(-1, BLOCK[kind])
    b, i = raw.long(), torch.arange(256, device="cuda")
    half = lambda at: raw[:, at:at + 2].contiguous().view(torch.float16).double()
    if kind == "Q4_K":
        g = i // 32
        sc = torch.where(g < 4, b[:, 4 + g % 4] & 63, (b[:, 12 + g % 4] & 15) + 16 * (b[:, 4 + g % 4] >> 6))
        mn = torch.where(g < 4, b[:, 8 + g % 4] & 63, (b[:, 12 + g % 4] >> 4) + 16 * (b[:, 8 + g % 4] >> 6))
        p = half(0) * (sc * ((b[:, 16 + 32 * (i // 64) + i % 32] >> (4 * (g % 2))) & 15))
        m = half(2) * mn
        return (p - m).view(rows, cols), (p + m).view(rows, cols)
    h, quarter, c = i // 128, i % 128 // 32, i % 32
    q = ((b[:, 64 * h + 32 * (quarter % 2) + c] >> (4 * (quarter // 2))) & 15) + 16 * (
        (b[:, 128 + 32 * h + c] >> (2 * quarter)) & 3) - 32
    sc = raw[:, 192:208].contiguous().view(torch.int8).long()[:, i // 16]
    w = half(208) * (sc * q)
    return w.view(rows, cols), w.abs().view(rows, cols)


def reference(raw, kinds, idx, w, x, experts, inter, width):
    out = torch.zeros(x.shape, dtype=F64, device="cuda")
    tol = torch.zeros_like(out)
    sizes = [(inter, width), (inter, width), (width, inter)]
    for e in range(experts):
        t, j = torch.nonzero(idx == e, as_tuple=True)
        if t.numel() == 0:
            continue
        step = [m * k // 256 * BLOCK[kind] for kind, (m, k) in zip(kinds, sizes)]
        (wg, ag), (wu, au), (wd, ad) = (decode(r[e * s:(e + 1) * s], kind, *mk)
                                        for r, s, kind, mk in zip(raw, step, kinds, sizes))
        xs = x[t].double()
        g, u = xs @ wg.T, xs @ wu.T
        dg, du = 2.0 ** -21 * (xs.abs() @ ag.T), 2.0 ** -21 * (xs.abs() @ au.T)
        s = g / (1 + torch.exp(-g))
        h = s * u
        dh = 1.1 * dg * u.abs() + s.abs() * du + 1.1 * dg * du + 2.0 ** -18 * h.abs()
        y, a = h @ wd.T, w[t, j].double()[:, None]
        dy = dh @ wd.abs().T + 2.0 ** -21 * (h.abs() @ ad.T)
        out.index_add_(0, t, a * y)
        tol.index_add_(0, t, a.abs() * (dy + 2.0 ** -22 * y.abs()))
    return out, tol


def pairs_of(mean, experts, g):
    """Ids of the pairs: some experts without any, one with more than two tiles, the others around `mean`."""
    few = torch.randint(0, 3, (experts,), generator=g) if mean == "one" else torch.randint(2, 11, (experts,), generator=g)
    few[3], few[experts - 2] = 0, 0
    few[experts // 2] = 19 if mean == "one" else 37
    return torch.repeat_interleave(torch.arange(experts), few)


@pytest.mark.parametrize("inter,width", [(512, 2048), (1024, 1024), (2048, 512)])
@pytest.mark.parametrize("kinds", [("Q4_K", "Q4_K", "Q4_K"), ("Q6_K", "Q6_K", "Q6_K"), ("Q6_K", "Q6_K", "Q4_K")])
@pytest.mark.parametrize("mean", ["one", "several"])
def test_many_turns_of_a_workgroup(mean, kinds, inter, width):
    experts = 131
    g = torch.Generator().manual_seed(inter + len(mean))
    gd = torch.Generator(device="cuda").manual_seed(inter + len(mean))
    ids = pairs_of(mean, experts, g)
    ids = ids[torch.randperm(ids.numel(), generator=g)]
    size = 8 if mean == "one" else 16
    # the launch takes small tiles for means of up to 1.5 (of 8 pairs) and 8 (of 16)
    assert (ids.numel() <= 1.5 * experts) if mean == "one" else (1.5 * experts < ids.numel() <= 8 * experts)
    tiles = sum(-(-n // size) for n in torch.bincount(ids, minlength=experts).tolist())
    for m, k, tall in ((inter, width, 16), (width, inter, 32)):
        waves = 8 if k > 1024 else 4 if k > 512 else 2          # that share a row's blocks
        assert tiles * (m // tall) * waves // 8 > 4 * 256        # turns: more than four a workgroup
    idx = ids.to(I32).view(-1, 1).cuda()
    w = (0.5 + torch.rand(idx.shape, generator=gd, device="cuda"))
    x = torch.randn((idx.shape[0], width), generator=gd, device="cuda")
    raw = [weights(gd, kind, experts * inter * width) for kind in kinds]
    order, starts = ops.moe_group_rows(idx, experts)
    out = torch.full_like(x, float("nan"))
    ops.moe_experts_rows(raw[0], raw[1], kinds[0], raw[2], kinds[2], experts, order, starts, w, x, inter, out=out)
    want, tol = reference(raw, kinds, idx, w, x, experts, inter, width)
    bad = ~((out.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.any(dim=1).sum()), float(((out.double() - want).abs() / tol).max()))
