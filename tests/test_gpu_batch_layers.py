"""Layers over many rows at once: the MoE layer's prefill against its decode step, the attention layer over a batch of
requests (projections, norm and rotation, paged 8-bit cache, attention, gate, projection) against its parts.

Tolerances. A row of K-quant products is an fp32 dot product: an error of 2^-21 of the sum of its terms' magnitudes, which
for random signs is some sqrt(K) of the sum's size (45 at K = 2048): below 2^-15 of the outputs' rms a product, so three in
a row (gate or up, down, combine; or the projection behind attention) stay below 1e-4 of the rms, of either path."""

from __future__ import annotations

import kv8_ref
import numpy as np
import pytest
import torch

from qwen35_hip import ops, synth
from qwen35_hip.decode_layers import AttnLayerBatch, AttnLayerDecode, MoeLayerDecode

pytestmark = pytest.mark.gpu
F32, I32 = np.float32, np.int32


def dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).cuda()


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


def q4(M, K, s):
    return dev(synth.q4k_table(M, K, seed_tensor=s))


def close(got, want, what):
    """Within 2e-4 of the rows' rms (1e-4 for each of two paths)."""
    rms = np.sqrt((want.astype(np.float64) ** 2).mean(axis=-1, keepdims=True))
    assert np.all(np.abs(got - want) <= 2e-4 * rms), (what, float((np.abs(got - want) / rms).max()))


@pytest.mark.parametrize("T", [1, 7, 50, 300])
def test_moe_prefill_equals_decode_steps(T):
    r = np.random.default_rng(T)
    dm, E, k, I, S = 512, 64, 8, 256, 512
    layer = MoeLayerDecode(q4(E, dm, 60), q4(E * I, dm, 61), q4(E * I, dm, 62), q4(E * dm, I, 63), q4(1, dm, 64), q4(S, dm, 65),
                           q4(S, dm, 66), q4(dm, S, 67), d_model=dm, experts=E, k=k, inter=I, shared=S)
    xs = dev((0.2 * r.standard_normal((T, dm))).astype(F32))
    got = host(layer.prefill(xs))
    want = np.stack([host(layer.forward(xs[t], torch.empty(dm, device="cuda"))) for t in range(T)])
    close(got, want, T)
    out = torch.empty_like(xs)
    assert layer.prefill(xs, out=out).data_ptr() == out.data_ptr() and np.array_equal(host(out), got)


def attn_layer(r, dm=512, h=8, kvh=2, hd=128, max_seq_len=8):
    ws = [q4(2 * h * hd, dm, 50), q4(kvh * hd, dm, 51), q4(kvh * hd, dm, 52), q4(dm, h * hd, 53)]
    qn, kn = (dev((1 + 0.1 * r.standard_normal(hd)).astype(F32)) for _ in range(2))
    return AttnLayerDecode(*ws, qn, kn, d_model=dm, heads=h, kv_heads=kvh, head_dim=hd, rope_dim=32, max_seq_len=max_seq_len)


def parts(a, x, pos):
    """Query, gate, key and value of one token by the one-token calls."""
    qg, k, v = (torch.empty(n, device="cuda") for n in (2 * a.qd, a.kd, a.kd))
    for name, y in (("qg", qg), ("k", k), ("v", v)):
        a._proj(name, x, y, a.dm)
    q, gate = ops.attn_split_qg(qg, a.h, a.hd)
    q, k = q.view(a.h, a.hd), k.view(a.kvh, a.hd)
    ops.attn_head_norm(q, a.q_norm, eps=a.eps)
    ops.attn_head_norm(k, a.k_norm, eps=a.eps)
    ops.rope_forward(q, pos, a.rope_dim, a.theta)
    ops.rope_forward(k, pos, a.rope_dim, a.theta)
    return [host(t) for t in (q, gate.view(a.h, a.hd), k, v.view(a.kvh, a.hd))]


def test_attention_batch_of_layers():
    """Three steps of four requests through two layers that share one plan a step: prompts, then single tokens and a second
    chunk, with padding rows. Keys and values in the cache are the one-token calls' within the codes' steps, the output that
    of 64-bit attention over the cache's codes."""
    r = np.random.default_rng(2)
    page, pages, rows, width = 16, 32, 60, 8
    layers = [attn_layer(r), attn_layer(r)]
    batch = [AttnLayerBatch(a, pages, page) for a in layers]
    table, free = torch.zeros((4, width), dtype=torch.int32, device="cuda"), dev(r.permutation(pages), I32)
    head, lens = torch.zeros(1, dtype=torch.int32, device="cuda"), np.zeros(4, int)
    known = [[([], []) for _ in range(4)] for _ in layers]   # keys and values so far, by layer and request
    for fresh in ([37, 1, 20, 0], [1, 1, 30, 2], [1, 1, 1, 1]):
        plan = ops.kv8_plan(dev(lens, I32), dev(fresh, I32), table, free, head, page, rows)
        head = plan[4]
        n = int(np.sum(fresh))
        xs = dev((0.5 * r.standard_normal((rows, layers[0].dm))).astype(F32))
        start = np.concatenate([[0], np.cumsum(fresh)])
        lens = lens + fresh
        for li, (a, b) in enumerate(zip(layers, batch)):
            got = host(b.forward(xs, table, plan))
            q, gate = np.zeros((2, n, a.h, a.hd), F32)
            for req in range(4):
                for i in range(start[req], start[req + 1]):
                    q[i], gate[i], k, v = parts(a, xs[i], int(lens[req] - start[req + 1] + i))
                    known[li][req][0].append(k)
                    known[li][req][1].append(v)
                if lens[req] == 0:
                    continue
                # A row of the cache is off by half a step of its page's scale, and by another half for each later rescaling
                # of the page: at most one a step of the batch. The scale is at most the largest value / 127.
                t = np.arange(lens[req])
                slots = host(table)[req, t // page] * page + t % page
                for w, cached in enumerate(ops.kv8_read_rows(b.cache, dev(slots, I32))):
                    want = np.stack(known[li][req][w])
                    step = np.abs(want).max() / 127
                    assert np.all(np.abs(host(cached) - want) <= (0.5 + 0.5 * 3 + 1e-3) * step)
            ref = kv8_ref.Cache(pages, a.kvh, page, a.hd)
            c = b.cache
            ref.codes = [host(c.k).astype(np.float64),
                         host(c.v).swapaxes(3, 4).reshape(pages, a.kvh, page, a.hd).astype(np.float64)]
            ref.scales = [host(c.k_scale).astype(np.float64), host(c.v_scale).astype(np.float64)]
            mid, _ = kv8_ref.attention(q, ref, host(table), start, lens, gate)
            w, M = a.w["out"]
            want = host(ops.matmul_rows(w, a.wtype, M * a.qd, dev(mid.reshape(n, a.qd), F32), M, a.qd))
            close(got[:n], want, (li, fresh))
            assert np.all(np.isfinite(got))


def test_a_step_of_both_layers_in_a_graph():
    """A planned step through an attention and a MoE layer, captured once and replayed over other lengths and rows with eager
    work between: every replay equals the eager step bit for bit."""
    r = np.random.default_rng(4)
    page, pages, rows, requests, width, dm, E, I, S = 16, 24, 20, 3, 6, 512, 16, 256, 512
    a = attn_layer(r)
    moe = MoeLayerDecode(q4(E, dm, 60), q4(E * I, dm, 61), q4(E * I, dm, 62), q4(E * dm, I, 63), q4(1, dm, 64), q4(S, dm, 65),
                         q4(S, dm, 66), q4(dm, S, 67), d_model=dm, experts=E, k=4, inter=I, shared=S)
    i32 = dict(dtype=torch.int32, device="cuda")
    free = dev(r.permutation(pages), I32)
    cached, fresh, xs = torch.zeros(requests, **i32), torch.zeros(requests, **i32), torch.zeros((rows, dm), device="cuda")

    class Side:
        def __init__(self):
            self.batch = AttnLayerBatch(a, pages, page)
            self.table, self.head = torch.zeros((requests, width), **i32), torch.zeros(1, **i32)

        def step(self):
            plan = ops.kv8_plan(cached, fresh, self.table, free, self.head, page, rows, free_head_out=self.head)
            return moe.prefill(self.batch.forward(xs, self.table, plan))

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
        xs.copy_(dev((0.5 * r.standard_normal((rows, dm))).astype(F32)))
        g.replay()
        torch.cuda.synchronize()
        want = eager.step()
        assert torch.equal(out, want), new
        assert torch.equal(captured.table, eager.table) and torch.equal(captured.head, eager.head)
        assert torch.equal(captured.batch.cache.k_scale, eager.batch.cache.k_scale)
        lens += new
