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
