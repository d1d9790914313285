"""Rows that the row kernels read in whole 16-byte pieces without a look at the operand's ends: no piece of theirs lies outside it."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def inner_rows(tmp_path_factory):
    work = tmp_path_factory.mktemp("rules")
    src, lib = work / "rules.cpp", work / "rules.so"
    src.write_text('#include "rules.h"\nextern "C" void inner_rows(long long rows, long long pitch, long long* out) {'
                   " const auto r = b200ait::inner_rows(rows, pitch); out[0] = r.begin, out[1] = r.end; }\n")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror", "-I", os.path.join(ROOT, "aitemplate_b200", "csrc"),
                    str(src), "-o", str(lib)], check=True)
    lib = ctypes.CDLL(str(lib))

    def call(rows, pitch):
        out = (ctypes.c_longlong * 2)()
        lib.inner_rows(ctypes.c_longlong(rows), ctypes.c_longlong(pitch), out)
        return out[0], out[1]

    return call


@pytest.mark.parametrize("gated", [1, 2])
@pytest.mark.parametrize("n", range(1, 20))
def test_pieces_of_inner_rows_lie_in_the_operand(inner_rows, n, gated):
    """A row of n elements from element `at` on, at `place` elements after a 16-byte boundary, is read from the boundary at or ahead of its
    start to the one at or behind its end."""
    for pitch in (n * gated, n * gated + 1, n * gated + 5):
        for rows in range(1, 21):
            begin, end = inner_rows(rows, pitch)
            size = (rows - 1) * pitch + n * gated
            for place in range(8):
                for row in range(max(begin, 0), min(end, rows)):
                    at = row * pitch
                    skew = (place + at) % 8
                    first, past = at - skew, at - skew + (n + skew + 7) // 8 * 8
                    assert 0 <= first and past <= size, (pitch, rows, place, row)


def test_most_rows_are_inner(inner_rows):
    """All but the first and the last one, where a pitch holds the elements that a piece takes along."""
    assert inner_rows(1000, 7) == (1, 999) and inner_rows(1000, 4096) == (1, 999)
    assert inner_rows(1000, 1) == (7, 993) and inner_rows(3, 1)[0] > inner_rows(3, 1)[1]
