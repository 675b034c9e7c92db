"""Arrays that overlap, refused before any launch, on the CPU. Pointers here are never followed."""

from __future__ import annotations

import pytest

from qwen35_hip import _lib

INV = _lib.STATUS_INVALID_ARGUMENT


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


BASE = 1 << 20


@pytest.mark.parametrize("idx,order,starts", [
    (BASE, BASE, 4 * BASE), (BASE, BASE + 4 * 1999, 4 * BASE), (BASE + 4 * 1999, BASE, 4 * BASE),   # the ids in place, or by one
    (BASE, 2 * BASE, BASE + 4 * 1999), (BASE, 2 * BASE, BASE - 4 * 16), (BASE, 2 * BASE, 2 * BASE + 8)])
def test_group(lib, idx, order, starts):
    assert lib.qwen_moe_group_rows(idx, 2000, 16, order, starts, None) == INV
    assert "overlap" in lib.qwen_last_error().decode()


@pytest.mark.parametrize("over", [
    dict(kv_len="cached"), dict(kv_len="fresh"), dict(row_start="cached"), dict(slots="free"), dict(pos="fresh"),
    dict(table="free"), dict(kv_len="head"), dict(head_out="cached"), dict(slots="cached", by=4 * 63), dict(table="fresh", by=-4)])
def test_plan(lib, over):
    """Lengths updated in place and the like: other workgroups of the call still read them."""
    at = {n: (i + 1) * BASE for i, n in enumerate(("cached", "fresh", "table", "free", "head", "head_out", "row_start", "kv_len",
                                                   "slots", "pos"))}
    (out, of), by = list(over.items())[0], over.get("by", 0)
    at[out] = at[of] + by
    assert lib.qwen_kv8_plan(at["cached"], at["fresh"], 64, at["table"], 32, at["free"], 900, at["head"], at["head_out"], 64, 2000,
                             at["row_start"], at["kv_len"], at["slots"], at["pos"], None) == INV
    assert "overlaps" in lib.qwen_last_error().decode()


@pytest.mark.parametrize("over", [dict(out="q"), dict(out="q", by=16), dict(out="q", by=-16), dict(out="gate", by=4096),
                                  dict(out="gate", by=-64)])
def test_attention(lib, over):
    """Rows written beside others that are still to be read."""
    at = dict(q=BASE, gate=2 * BASE, out=3 * BASE)
    (out, of), by = list(over.items())[0], over.get("by", 0)
    at[out] = at[of] + by
    C = 4 * BASE
    assert lib.qwen_attn_kv8_rows(at["q"], C, C, C, C, 8, 64, C, 4, C, C, 2, at["gate"], at["out"], 3, 16, 2, 256, C, 1 << 40,
                                  None) == INV
    assert "overlaps" in lib.qwen_last_error().decode()
