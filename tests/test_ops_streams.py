"""Memory that a call with `stream=` allocates: it belongs to that stream, not to the current one."""

from __future__ import annotations

import ast
import contextlib
import inspect

import numpy as np
import pytest
import torch

from qwen35_hip import ops


# ------------------------------------------------------------------ on the CPU
def test_no_call_with_a_stream_allocates_on_the_current_one():
    """Every function of ops with a `stream` takes its memory from the helpers that know it."""
    tree = ast.parse(inspect.getsource(ops))
    helpers = ("_empty", "_like", "_scratch")
    seen = 0
    for f in tree.body:
        if not isinstance(f, ast.FunctionDef) or "stream" not in [a.arg for a in f.args.args] or f.name in helpers:
            continue
        for call in (c for c in ast.walk(f) if isinstance(c, ast.Call)):
            name = ast.unparse(call.func)
            assert not name.startswith(("torch.empty", "torch.zeros", "torch.full")), f"{f.name}: {name}"
            if name in helpers:
                seen += 1
                assert ast.unparse(call.args[0]) == "stream", f"{f.name}: {ast.unparse(call)}"
    assert seen > 50


def test_helpers_allocate_under_the_stream(monkeypatch):
    """Under it where one is given, and an output (not a workspace) marked as used by the current one."""
    at, made, recorded = [None], [], []
    empty = torch.empty

    @contextlib.contextmanager
    def under(s):
        at.append(s)
        yield
        at.pop()

    def counted(*a, **k):
        made.append(at[-1])
        return empty(*a, **k)

    monkeypatch.setattr(torch.cuda, "stream", under)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: "now")
    monkeypatch.setattr(torch, "empty", counted)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: recorded.append(s))
    like = empty((2, 3), dtype=torch.bfloat16)
    for s in ("other", None):
        made.clear(), recorded.clear()
        t = [ops._empty(s, (4, 5), "cpu", torch.int32), ops._scratch(s, 3, "cpu"), ops._like(s, like)]
        assert [tuple(x.shape) for x in t] == [(4, 5), (16,), (2, 3)]
        assert [x.dtype for x in t] == [torch.int32, torch.uint8, torch.bfloat16]
        assert made == ([s] * 3 if s else [None] * 2) and recorded == (["now"] * 2 if s else [])


# ------------------------------------------------------------------ on the GPU
def dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).cuda()


def attention_call(r):
    cache = ops.kv8_cache(40, 2, 128, 16)
    k, v = (dev(r.standard_normal((600, 2, 128)), np.float32) for _ in range(2))
    ops.kv8_store_rows(k, v, torch.arange(600, dtype=torch.int32, device="cuda"), cache)
    q = dev(r.standard_normal((40, 16, 128)), np.float32)
    args = (q, cache, torch.arange(38, dtype=torch.int32, device="cuda").view(1, -1), dev([0, 40], np.int32),
            dev([600], np.int32))
    return lambda **kw: ops.attn_kv8_rows(*args, **kw), ops.attn_kv8_workspace_bytes(40, 1, 16, 2, 128)


def experts_call(r):
    rows, top, experts, width, inter = 40, 4, 8, 512, 256
    raw = []
    for _ in range(3):
        b = r.integers(0, 256, (experts * inter * width // 256, 144), dtype=np.uint8)
        b[:, :4] = np.array([1e-4, 7e-4], np.float16).view(np.uint8)
        raw.append(dev(b.reshape(-1)))
    idx = dev(np.stack([r.permutation(experts)[:top] for _ in range(rows)]), np.int32)
    w, x = dev(r.uniform(0, 1, (rows, top)), np.float32), dev(r.standard_normal((rows, width)), np.float32)
    order, starts = ops.moe_group_rows(idx, experts)
    return (lambda **kw: ops.moe_experts_rows(raw[0], raw[1], "Q4_K", raw[2], "Q4_K", experts, order, starts, w, x, inter, **kw),
            ops.moe_experts_rows_workspace_bytes(rows, top, experts, width, inter))


@pytest.mark.gpu
@pytest.mark.parametrize("make", [attention_call, experts_call])
def test_memory_of_a_call_on_another_stream(make):
    """A call on a stream that is still busy: tensors of the workspace's and the output's size that the current stream makes
    and fills at once afterwards are not the call's; and an output read on the current stream and dropped there is not
    handed to the stream's next call before it has been read."""
    call, ws_bytes = make(np.random.default_rng(1))
    want = call()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(3):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            torch.cuda._sleep(10_000_000)
        got = call(stream=s)
        others = [torch.full((n,), 0x7f, dtype=torch.uint8, device="cuda") for n in (ws_bytes, max(ws_bytes, 16), want.numel() * 4)]
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        assert all(bool((t == 0x7f).all()) for t in others)
        torch.cuda._sleep(10_000_000)
        copy = got.clone()           # on the current stream, behind the wait above
        del got, others
        again = call(stream=s, out=None)
        again.record_stream(s)
        with torch.cuda.stream(s):
            again.zero_()
        torch.cuda.synchronize()
        assert torch.equal(copy, want)
