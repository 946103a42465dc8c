"""The integer arithmetic that bounds the linear attention's accesses (csrc/segments.h), compiled for the CPU and checked
against Python's integers over offsets that hold anything."""

import ctypes
import random
import subprocess
from pathlib import Path

import pytest

HEADER = Path(__file__).resolve().parent.parent / "ez-ops_amd" / "csrc" / "segments.h"
SOURCE = """
#include "%s"
extern "C" void seq_rows(int begin, int end, int T, int max_q, int* out) {
  const ez::SeqRows r = ez::seq_rows(begin, end, T, max_q);
  out[0] = r.first; out[1] = r.count;
}
"""
MIN, MAX = -(1 << 31), (1 << 31) - 1


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("segments")
    (d / "s.cpp").write_text(SOURCE % HEADER)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", str(d / "s.cpp"), "-o",
                    str(d / "s.so")], check=True, timeout=60)
    return ctypes.CDLL(str(d / "s.so"))


def test_rows_of_a_sequence_stay_in_the_tensors(lib):
    """Ends near the lowest integer behind a begin > 0, ends and begins past the rows, offsets that decrease."""
    got = (ctypes.c_int * 2)()
    r = random.Random(1)
    ends = [MIN, MIN + 1, MIN + 40, -41, -1, 0, 1, 39, 40, 41, 99, 100, 101, 1 << 30, MAX]
    cases = [(b, e, T, q) for b in ends for e in ends for T in (1, 100, (1 << 30) - 1) for q in (1, 40, T)]
    cases += [(r.randint(MIN, MAX), r.randint(MIN, MAX), t, r.randint(1, t)) for t in
              (r.randint(1, (1 << 30) - 1) for _ in range(2000))]
    for b, e, T, q in cases:
        lib.seq_rows(b, e, T, q, got)
        first, end = min(max(b, 0), T), min(max(e, 0), T)
        n = min(end - first, q)
        if n > 0:
            assert list(got) == [first, n], (b, e, T, q, list(got))
        else:
            assert got[1] <= 0, (b, e, T, q, list(got))
        assert 0 <= got[0] <= T and (got[1] <= 0 or got[0] + got[1] <= T), (b, e, T, q, list(got))
