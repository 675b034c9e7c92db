"""The attention layer over a batch of requests with the 4-bit cache and positions of several axes: norm and rotation, store
and attention as they are used together.

Tolerances. Rows of products as in the layers over many rows: 1e-4 of the rows' rms for each path. A number in the cache is off
by half a step of its group beside that, its group's step as the cache holds it (a number rounds to the nearest code, and the
least number and 15 steps reach over the group)."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from qwen35_hip import ops, synth
from qwen35_hip.decode_layers import AttnLayerBatch, AttnLayerDecode

gpu = pytest.mark.gpu
F32, F64, I32 = np.float32, np.float64, np.int32


def test_refusals():
    layer = SimpleNamespace(rope_dim=32, kvh=2, hd=128, q_norm=torch.ones(128))
    for bits in (0, 2, 16, "4"):
        with pytest.raises(ValueError, match="cache_bits"):
            AttnLayerBatch(layer, 4, cache_bits=bits)
    for sections in ((16, 16), (8,), ()):
        with pytest.raises(ValueError, match="rope_sections"):
            AttnLayerBatch(layer, 4, rope_sections=sections)
    xs, plan = torch.empty((3, 512)), [None] * 5
    for sections, positions in ((None, torch.zeros((1, 3), dtype=torch.int32)), ((8, 8), None)):
        batch = object.__new__(AttnLayerBatch)   # without a cache, which is a device's
        batch.layer, batch.sections = layer, sections
        with pytest.raises(ValueError, match="positions"):
            batch.forward(xs, None, plan, positions=positions)


def dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).cuda()


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


def layer_of(r, dm=512, h=8, kvh=2, hd=128):
    q4 = lambda M, K, s: dev(synth.q4k_table(M, K, seed_tensor=s))
    ws = [q4(2 * h * hd, dm, 50), q4(kvh * hd, dm, 51), q4(kvh * hd, dm, 52), q4(dm, h * hd, 53)]
    qn, kn = (dev((1 + 0.1 * r.standard_normal(hd)).astype(F32)) for _ in range(2))
    return AttnLayerDecode(*ws, qn, kn, d_model=dm, heads=h, kv_heads=kvh, head_dim=hd, rope_dim=32, max_seq_len=8)


def rotated(x, pos, axis, theta):
    """x [heads, dim] in 64 bits, pos of each axis."""
    half = len(axis)
    angle = np.array([pos[a] for a in axis], F64) * theta ** (-np.arange(half) / half)
    y, a, b = x.astype(F64), x[:, :half].astype(F64), x[:, half:2 * half].astype(F64)
    y[:, :half], y[:, half:2 * half] = a * np.cos(angle) - b * np.sin(angle), b * np.cos(angle) + a * np.sin(angle)
    return y


def parts(a, x, pos, axis):
    """Query, gate, key and value of one token: projections and norm by the one-token calls, the rotation by its formula."""
    qg, k, v = (torch.empty(n, device="cuda") for n in (2 * a.qd, a.kd, a.kd))
    for name, y in (("qg", qg), ("k", k), ("v", v)):
        a._proj(name, x, y, a.dm)
    q, gate = ops.attn_split_qg(qg, a.h, a.hd)
    q, k = q.view(a.h, a.hd), k.view(a.kvh, a.hd)
    ops.attn_head_norm(q, a.q_norm, eps=a.eps)
    ops.attn_head_norm(k, a.k_norm, eps=a.eps)
    return (rotated(host(q), pos, axis, a.theta), host(gate.view(a.h, a.hd)).astype(F64), rotated(host(k), pos, axis, a.theta),
            host(v.view(a.kvh, a.hd)))


AXES = {None: [0] * 16, (6, 5, 5): [0, 1, 2] * 5 + [0], (10, 6): [0] * 10 + [1] * 6}


@gpu
@pytest.mark.parametrize("sections,bits,page", [((6, 5, 5), 4, 16), ((10, 6), 4, 64), (None, 4, 8), ((6, 5, 5), 8, 16)])
def test_steps_of_a_batch(sections, bits, page):
    """Three steps of four requests: prompts, then single tokens and a second chunk, with padding rows."""
    r = np.random.default_rng(2)
    pages, rows, width = 512 // page, 60, 128 // page
    a = layer_of(r)
    turns = sections != (10, 6)
    b = AttnLayerBatch(a, pages, page, cache_bits=bits, rope_sections=sections, rope_interleaved=turns)
    table, free = torch.zeros((4, width), dtype=torch.int32, device="cuda"), dev(r.permutation(pages), I32)
    head, lens = torch.zeros(1, dtype=torch.int32, device="cuda"), np.zeros(4, int)
    known = [([], []) for _ in range(4)]
    axis = AXES[sections]
    for fresh in ([37, 1, 20, 0], [1, 1, 30, 2], [1, 1, 1, 1]):
        plan = ops.kv8_plan(dev(lens, I32), dev(fresh, I32), table, free, head, page, rows)
        head = plan[4]
        n = int(np.sum(fresh))
        start = np.concatenate([[0], np.cumsum(fresh)])
        xs = dev((0.5 * r.standard_normal((rows, a.dm))).astype(F32))
        positions = None
        if sections:
            positions = r.integers(0, 300, (len(sections), rows)).astype(I32)
        got = host(b.forward(xs, table, plan, positions=None if positions is None else dev(positions)))
        assert np.all(np.isfinite(got))
        mid = np.zeros((n, a.h, a.hd))
        lens = lens + fresh
        for req in range(4):
            if fresh[req] == 0:
                continue
            t = np.arange(lens[req])
            slots = dev(host(table)[req, t // page] * page + t % page, I32)
            toks = []
            for i in range(start[req], start[req + 1]):
                at = int(lens[req] - start[req + 1] + i)
                toks.append(parts(a, xs[i], positions[:, i] if sections else [at], axis))
                known[req][0].append(toks[-1][2])
                known[req][1].append(toks[-1][3])
            if bits == 4:
                cached = [host(x).astype(F64) for x in ops.kv4_read_rows(b.cache, slots)]
                p, o = host(slots) // page, host(slots) % page
                ks = host(b.cache.k_scale.float())[p, :, o // 8, :, o % 8]
                steps = np.repeat(ks, 64, axis=-1), host(b.cache.v_scale.float())[p, :, o][..., None]
                for have, want, step in zip(cached, known[req], steps):
                    want = np.stack(want).astype(F64)
                    rms = np.sqrt((want ** 2).mean(-1, keepdims=True))
                    assert np.all(np.abs(have - want) <= 0.5 * step + 2e-4 * rms)
            else:
                cached = [host(x).astype(F64) for x in ops.kv8_read_rows(b.cache, slots)]
            k, v = cached
            for i, (q, gate, _, _) in enumerate(toks):
                seen = int(lens[req]) - len(toks) + i + 1
                for h in range(a.h):
                    g = h // (a.h // a.kvh)
                    s = k[:seen, g] @ q[h] / np.sqrt(a.hd)
                    e = np.exp(s - s.max())
                    mid[start[req] + i, h] = e / e.sum() @ v[:seen, g] / (1 + np.exp(-gate[h]))
        w, M = a.w["out"]
        want = host(ops.matmul_rows(w, a.wtype, M * a.qd, dev(mid.reshape(n, a.qd), F32), M, a.qd))
        rms = np.sqrt((want.astype(F64) ** 2).mean(axis=-1, keepdims=True))
        assert np.all(np.abs(got[:n] - want) <= 2e-4 * rms), float((np.abs(got[:n] - want) / rms).max())


@gpu
def test_a_step_in_a_graph():
    """A planned step captured once and replayed over other lengths, rows and positions with eager work between: every replay
    equals the eager step bit for bit, and so do the caches."""
    r = np.random.default_rng(4)
    page, pages, rows, requests, width = 16, 24, 20, 3, 6
    a = layer_of(r)
    i32 = dict(dtype=torch.int32, device="cuda")
    free = dev(r.permutation(pages), I32)
    cached, fresh, xs = torch.zeros(requests, **i32), torch.zeros(requests, **i32), torch.zeros((rows, a.dm), device="cuda")
    positions = torch.zeros((3, rows), **i32)

    class Side:
        def __init__(self):
            self.batch = AttnLayerBatch(a, pages, page, cache_bits=4, rope_sections=(6, 5, 5))
            self.table, self.head = torch.zeros((requests, width), **i32), torch.zeros(1, **i32)

        def step(self):
            plan = ops.kv8_plan(cached, fresh, self.table, free, self.head, page, rows, free_head_out=self.head)
            return self.batch.forward(xs, self.table, plan, positions=positions)

    eager, captured = Side(), Side()
    for side in (eager, captured):
        side.step()   # idle requests: loads the kernels, takes no page
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = captured.step()
    lens = np.zeros(requests, int)
    for new in ([11, 0, 3], [1, 6, 1], [1, 1, 18], [1, 1, 1]):
        cached.copy_(dev(lens, I32))
        fresh.copy_(dev(new, I32))
        xs.copy_(dev((0.5 * r.standard_normal((rows, a.dm))).astype(F32)))
        positions.copy_(dev(r.integers(0, 5000, (3, rows)), I32))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager.step()), new
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(captured.batch.cache, eager.batch.cache)
                   if torch.is_tensor(x))
        lens += new


@gpu
def test_no_rows():
    a = layer_of(np.random.default_rng(0))
    i32 = dict(dtype=torch.int32, device="cuda")
    b = AttnLayerBatch(a, 8, 16, cache_bits=4, rope_sections=(8, 8))
    for requests in (0, 2):
        table, none = torch.zeros((requests, 4), **i32), torch.zeros(requests, **i32)
        plan = ops.kv8_plan(none, none, table, torch.arange(3, **i32), torch.zeros(1, **i32), 16, 0)
        assert b.forward(torch.empty((0, a.dm), device="cuda"), table, plan, positions=torch.zeros((2, 0), **i32)).shape == (0, a.dm)
