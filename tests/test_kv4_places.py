"""Where the 4-bit attention's pieces lie in its workspace (csrc/kv4_places.hpp), walked on the host: an entry that the join takes,
whatever it holds, names places of the workspace alone, and every entry that a call writes is taken."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "qwen-3.5-cuda_amd" / "csrc"
SHIM = """
#include "kv4_places.hpp"
extern "C" int joinable(int first, int pieces, int split, int all) { return qk::joinable(first, pieces, split, all); }
extern "C" int place(int first, int split, int piece) { return qk::places_of(first, split).of(piece); }
"""
ROWS, FILL, WIDE = 8, 256, 128
REGION = FILL * WIDE


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    d = tmp_path_factory.mktemp("places")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", f"-I{CSRC}", "-o", str(d / "shim.so"), str(d / "shim.cpp")],
                   check=True)
    return ctypes.CDLL(str(d / "shim.so"))


@pytest.mark.parametrize("split", [8 * 520, 8 * 1032, 8 * 2400])
@pytest.mark.parametrize("regions", [0, 2])
def test_what_is_joined_lies_in_the_workspace(rule, split, regions):
    all_places = split + regions * REGION
    borders = (0, split, split + REGION, split + 2 * REGION)
    firsts = {b + d for b in borders for d in (*range(-260, 260, 13), -129, -128, -127, -9, -8, -7, -1, 0, 1, 7, 8, 127, 128)}
    for first in sorted(firsts) + [2 ** 31 - 1, -(2 ** 31), 1 << 30, split // 2, split + REGION // 2]:
        for pieces in (*range(-2, 40), 100, 255, 256, 257, 511, split // ROWS - 1, split // ROWS, split // ROWS + 1, 1 << 20,
                       2 ** 31 - 1, -(2 ** 31)):
            if rule.joinable(first, pieces, split, all_places):
                assert pieces > 1
                low, high = (0, split) if first < split else (split, all_places)
                for p in {0, 1, pieces // 2, pieces - 1}:
                    assert low <= rule.place(first, split, p) < high, (first, pieces, p)


def test_entries_that_calls_write_are_joined(rule):
    split = ROWS * 700
    for row in (0, 3, 7):
        for item in (0, 1, 350, 698):
            for pieces in range(2, 700 - item + 1):
                assert rule.joinable(item * ROWS + row, pieces, split, split)
            assert not rule.joinable(item * ROWS + row, 700 - item + 1, split, split)
    for row in (0, 31, 127):
        for group in (0, 1, 128, 254):
            for pieces in range(2, FILL - group + 1):
                assert rule.joinable(split + group * WIDE + row, pieces, split, split + 2 * REGION)
                assert not rule.joinable(split + group * WIDE + row, pieces, split, split)   # a workspace without room for them
