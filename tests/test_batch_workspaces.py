"""Workspace sizes of the operators of several requests: one sized for a server's largest step serves every smaller one."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from qwen35_hip import _lib, ops


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


ROWS = [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 31, 32, 33, 40, 63, 64, 65, 100, 127, 128, 129, 200, 256, 257, 512, 1000, 1024, 1025,
        2048, 4095, 4096, 5000, 20000]


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 2, 256), (1, 1, 64), (12, 12, 64), (24, 8, 128), (40, 1, 128), (31, 1, 64),
                                                (64, 2, 256), (33, 1, 64)])
def test_attention_workspace_serves_smaller_steps(lib, heads, kv_heads, dim):
    """Never more for fewer rows or fewer requests."""
    requests = [n for n in ROWS if n <= 4096]
    size = np.array([[lib.qwen_attn_kv8_workspace_bytes(r, b, heads, kv_heads, dim) for b in requests] for r in ROWS])
    assert (size > 0).all()
    assert (np.diff(size, axis=0) >= 0).all(), [ROWS[i] for i in np.argwhere(np.diff(size, axis=0) < 0)[0][:1]]
    assert (np.diff(size, axis=1) >= 0).all(), [requests[i] for i in np.argwhere(np.diff(size, axis=1) < 0)[0][1:]]


@pytest.mark.parametrize("experts,top,width,inter", [(256, 8, 2048, 512), (60, 4, 2048, 512), (1024, 1, 256, 256), (8, 2, 512, 256),
                                                     (1, 1, 2304, 256)])
def test_experts_workspace_serves_smaller_steps(lib, experts, top, width, inter):
    """Never more for fewer rows, across the sizes of tiles too."""
    size = np.array([lib.qwen_moe_experts_rows_workspace_bytes(r, top, experts, width, inter) for r in range(1, 9000)])
    assert (size > 0).all() and (np.diff(size) >= 0).all(), int(np.argmax(np.diff(size) < 0)) + 1


@pytest.mark.parametrize("rows,top,experts,width,inter,words", [
    (3, 8, 0, 512, 256, "experts"), (3, 8, 1025, 512, 256, "experts"), (3, 8, 2000, 512, 256, "experts"),
    (3, 8, 16, (1 << 20) + 256, 256, "2^20"), (3, 8, 16, 512, (1 << 20) + 256, "2^20"), (3, 8, 16, 500, 256, "256"),
    (3, 8, 16, 512, 0, "256"), (3, 0, 16, 512, 256, "picks"), (-1, 8, 16, 512, 256, "picks"), (1 << 22, 8, 16, 512, 256, "picks"),
    (1 << 21, 8, 16, 512, 1024, "one call"), (1 << 15, 1, 16, 1 << 19, 256, "one call")])
def test_experts_workspace_of_refused_sizes(lib, rows, top, experts, width, inter, words):
    """0, and the message of the call itself."""
    assert lib.qwen_moe_experts_rows_workspace_bytes(rows, top, experts, width, inter) == 0
    P = 1 << 20
    said = lib.qwen_last_error().decode()
    assert words in said
    assert lib.qwen_moe_experts_rows(P, P, 12, P, 12, experts, P, P, P, top, P, rows, width, inter, 2 * P, P, 1 << 60,
                                     None) == _lib.STATUS_INVALID_ARGUMENT
    assert lib.qwen_last_error().decode() == said


@pytest.mark.gpu
def test_attention_workspace_of_a_larger_step():
    """Requests leave while the step keeps its padded rows: the same workspace, and what a call of its own size gives."""
    r = np.random.default_rng(0)
    heads, kvh, dim, rows = 16, 2, 128, 64
    cache = ops.kv8_cache(rows, kvh, dim, 16)
    cache.k.copy_(torch.from_numpy(r.integers(-127, 128, tuple(cache.k.shape), dtype=np.int8)))
    cache.v.copy_(torch.from_numpy(r.integers(-127, 128, tuple(cache.v.shape), dtype=np.int8)))
    cache.k_scale.fill_(0.02), cache.v_scale.fill_(0.02)
    i32 = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()
    q = torch.from_numpy(r.standard_normal((rows, heads, dim)).astype(np.float32)).cuda()
    table, lens = np.arange(rows).reshape(rows, 1), r.integers(1, 17, rows)
    ws = torch.empty(ops.attn_kv8_workspace_bytes(rows, rows, heads, kvh, dim), dtype=torch.uint8, device="cuda")
    for n in (64, 63, 40, 1):
        ws.fill_(0x7f)
        args = (q, cache, i32(table[:n]), i32(np.arange(n + 1)), i32(lens[:n]))
        outs = [torch.zeros_like(q) for _ in range(2)]
        ops.attn_kv8_rows(*args, workspace=ws, out=outs[0])
        ops.attn_kv8_rows(*args, out=outs[1])
        assert torch.equal(*outs) and bool(outs[0][:n].any()) and not bool(outs[0][n:].any())
