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
