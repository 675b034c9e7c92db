"""Rotation by positions of several axes over more rows than one axis of a grid has threads for."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from qwen35_hip import ops
from test_gpu_mrope import dev, expected

pytestmark = pytest.mark.gpu
F32, I32 = np.float32, np.int32


@pytest.mark.parametrize("rows,heads,hd,sections,shift", [
    ((1 << 24) + 5, 1, 2, (1,), 0), (1 << 23, 3, 6, (1, 0, 1), 0),   # a workgroup a row and head
    ((1 << 24) + 1, 1, 64, (8, 8), 1),                               # and for heads that begin off 16 bytes
    ((1 << 26) + 5, 1, 64, (8, 8), 0),                               # a wave for some heads of a row
])
def test_rows_past_two_to_the_32_threads(rows, heads, hd, sections, shift):
    """Rows at both ends and between against the formula; every other row holds ones, whose rotation keeps a pair's length."""
    r = np.random.default_rng(hd)
    at = np.unique(np.concatenate([[0, 1, rows - 2, rows - 1], r.integers(0, rows, 40),
                                   np.arange(-3, 4) + min(rows - 4, (1 << 26 if hd == 64 and not shift else 1 << 24) // heads)]))
    at = at[at < rows]
    x = r.standard_normal((len(at), heads, hd)).astype(F32)
    pos = r.integers(0, 40000, (len(sections), len(at))).astype(I32)
    w = np.ones(hd, F32)
    memory = torch.ones(rows * heads * hd + shift, device="cuda")
    q = memory[shift:].view(rows, heads, hd)
    q[dev(at)] = dev(x)
    where = torch.zeros((len(sections), rows), dtype=torch.int32, device="cuda")
    where[:, dev(at)] = dev(pos)
    none = torch.empty((rows, 0, hd), device="cuda")
    ops.attn_qk_norm_mrope_rows(q, none, dev(w), dev(w), where, sections)
    torch.cuda.synchronize()
    want, tol = expected(x, w, pos, sections, True, 1e7, float(F32(1e-6)))
    assert np.all(np.abs(q[dev(at)].cpu().numpy() - want) <= tol)
    q[dev(at)] = 1.0   # position 0 turns by nothing: ones over their rms, sqrt(1 + 1e-6), and the norm's own 2^-20
    assert float((q - 1.0).abs_().max()) <= 5.1e-7 + 2.0 ** -20
