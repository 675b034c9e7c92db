"""Rows that see thousands of keys in one go, as a call of many prompts gives them to the 4-bit attention: their sums keep what an
fp32 evaluation keeps.

260 chunks of 70 rows over the same pages, too many to be cut, so that a row's tiles of 32 keys are summed one after the other."""

from __future__ import annotations

import numpy as np
import pytest

import kv4_ref
from qwen35_hip import ops
from test_gpu_kv4 import close, dev, gpu_cache, host, random_cache, tables

pytestmark = pytest.mark.gpu
F32, I32 = np.float32, np.int32
CHUNKS, ROWS, HEADS, DIM, PAGE = 260, 70, 2, 64, 64


def outputs(r, ref, table, total, sigma, some=24):
    """-> outputs of some random rows, their 64-bit form and its tolerance."""
    q = (sigma * r.standard_normal((CHUNKS * ROWS, HEADS, DIM))).astype(F32)
    got = host(ops.attn_kv4_rows(dev(q), gpu_cache(ref), dev(np.repeat(table, CHUNKS, 0)),
                                 dev(np.arange(CHUNKS + 1) * ROWS, I32), dev(np.full(CHUNKS, total), I32)))
    rows = r.choice(len(q), some, replace=False)
    return got[rows], *kv4_ref.attention(q[rows], ref, np.repeat(table, some, 0), range(some + 1),
                                         (total - ROWS + rows % ROWS + 1).tolist())


@pytest.mark.parametrize("total", [700, 3000, 12000])
def test_means_of_values_of_either_sign(total):
    """Weights of like size over values of mean zero: an output is small beside the sum of its terms' sizes, and each of the
    4 additions a tile to a sum of its own size rounds by 2^-24 of it at most, one way or the other. With 2^-20 for what does
    not grow (weights, products, exponentials) the root mean square is below (2^-20 + sqrt(4 tiles) 2^-24) of the outputs'."""
    r = np.random.default_rng(total)
    table, pages = tables(r, [total], PAGE)
    ref = random_cache(r, pages, HEADS, PAGE, DIM)
    ref.scale[1][:], ref.low[1][:] = 0.125, -7.5 * 0.125   # symmetric about 0
    got, want, _ = outputs(r, ref, table, total, 0.5)
    rms = lambda x: float(np.sqrt((x ** 2).mean()))
    assert rms(got - want) <= (2.0 ** -20 + np.sqrt(total / 8) * 2.0 ** -24) * rms(want)


@pytest.mark.parametrize("total", [3000, 12000, 40000])
@pytest.mark.parametrize("scale", [0.125, 0.111328125, 0.140625, 0.1015625])
def test_equal_weights(total, scale):
    """Queries of zeros: every key has the same weight, so that every addition to a row's sum of weights is of the same number
    and rounds the same way. Values above zero, whose sums err by as much as they are large."""
    r = np.random.default_rng(total)
    table, pages = tables(r, [total], PAGE)
    ref = random_cache(r, pages, HEADS, PAGE, DIM)
    ref.scale[1][:], ref.low[1][:] = scale, 1.0
    got, want, tol = outputs(r, ref, table, total, 0.0, some=8)
    close(got, want, tol)
