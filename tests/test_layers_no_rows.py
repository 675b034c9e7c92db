"""Steps without rows: what runs many rows at once takes none of them too."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from qwen35_hip import _lib, ops, synth
from qwen35_hip.decode_layers import AttnLayerBatch, AttnLayerDecode, MoeLayerDecode


def test_matmul_rows_multi_of_no_rows():
    """As matmul_rows of none: outputs may be null, everything else is still checked. Pointers here are never followed."""
    lib = _lib.load()
    call = lambda rows, y, w=1 << 20, M=256: lib.qwen_matmul_rows_multi(ctypes.cast((ops.GemvDesc * 1)(ops.GemvDesc(
        w, 12, M, 256 * 256, 0, y, 0)), ctypes.c_void_p), 1, None, rows, 256, None, 0, None)
    assert call(0, None) == _lib.STATUS_OK and call(0, 1 << 20) == _lib.STATUS_OK
    assert call(1, None) == _lib.STATUS_INVALID_ARGUMENT and call(-1, 1 << 20) == _lib.STATUS_INVALID_ARGUMENT
    assert call(0, None, w=None) == _lib.STATUS_INVALID_ARGUMENT and call(0, None, M=257) != _lib.STATUS_OK


@pytest.mark.gpu
def test_layers_of_no_rows():
    q4 = lambda M, K, s: torch.from_numpy(synth.q4k_table(M, K, seed_tensor=s)).cuda()
    dm, E, I, S = 512, 16, 256, 512
    moe = MoeLayerDecode(q4(E, dm, 60), q4(E * I, dm, 61), q4(E * I, dm, 62), q4(E * dm, I, 63), q4(1, dm, 64), q4(S, dm, 65),
                         q4(S, dm, 66), q4(dm, S, 67), d_model=dm, experts=E, k=4, inter=I, shared=S)
    xs = torch.empty((0, dm), device="cuda")
    assert moe.prefill(xs).shape == (0, dm)
    norm = torch.ones(128, device="cuda")
    attn = AttnLayerDecode(q4(2 * 8 * 128, dm, 50), q4(256, dm, 51), q4(256, dm, 52), q4(dm, 8 * 128, 53), norm, norm.clone(),
                           d_model=dm, heads=8, kv_heads=2, head_dim=128, rope_dim=32, max_seq_len=8)
    batch = AttnLayerBatch(attn, 8, 16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    for requests in (0, 2):
        table = torch.zeros((requests, 4), dtype=torch.int32, device="cuda")
        none = torch.zeros(requests, dtype=torch.int32, device="cuda")
        plan = ops.kv8_plan(none, none, table, i32(1, 2, 3), i32(0), 16, 0)
        assert batch.forward(xs, table, plan).shape == (0, dm)
        assert np.array_equal(plan[4].cpu(), [0])
