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
extern "C" int ws_slots(int segments, int T, int seg_sh) { return int(ez::ws_slots(segments, T, seg_sh)); }
extern "C" int ws_first(int first, int b, int seg_sh, int segments, int T) {
  return ez::ws_first(first, b, seg_sh, ez::ws_by_row(segments, T, seg_sh));
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


def _size(B, T, H, Hkv, D, mq=0):
    from ezops import _hip

    return _hip.lib().ezops_linear_attn_prefill_workspace_size(B, T, H, Hkv, D, mq)


def test_workspace_does_not_grow_with_the_batch():
    """States between the segments of long sequences alone: a bound of 2048 states of a kv head whatever the batch, and
    the same bytes for one long sequence beside 200 single tokens and beside 60000."""
    state = lambda D: D * D * 4  # noqa: E731
    r = random.Random(2)
    shapes = [(257, 2304, 32, 32, 128, 2048), (4096, 4096, 32, 32, 128, 0), (65536, 65536, 8, 8, 64, 0),
              (256, 8447, 32, 32, 128, 8192), (1, 1 << 24, 16, 16, 128, 0)]
    shapes += [(r.randint(1, 65536), int(2 ** r.uniform(0, 24)), h * g, h, r.choice((64, 128)), r.choice((0, 65, 1000)))
               for h, g in ((r.choice((1, 2, 3, 8, 32)), r.choice((1, 2, 4, 8, 16))) for _ in range(3000))]
    for s in shapes:
        assert _size(*s) <= 2048 * state(s[4]), (s, _size(*s) / state(s[4]))
    assert _size(200, 70000, 32, 32, 128) == _size(60000, 70000, 32, 32, 128) > 0


def test_workspace_slots_are_apart(lib):
    """Random ragged batches, cut by a length bound or not: the segments of every cut sequence have slots of their own
    inside the workspace, and so they do with offsets that decrease (inside it)."""
    r = random.Random(3)
    for _ in range(4000):
        sh, T, B = r.randint(6, 9), r.randint(65, 6000), r.randint(1, 40)
        seg, mq = 1 << sh, r.choice((0, 70, 130, 1000)) or T
        segments = (T >> sh) + B
        cu = sorted(r.choice((r.randint(0, T), 0, T)) for _ in range(B + 1))
        order = r.random() < 0.9
        if not order:
            r.shuffle(cu)
        slots = lib.ws_slots(segments, T, sh)
        assert slots <= segments and slots <= 2 * T // seg
        seen = set()
        for b in range(B):
            n = min(cu[b + 1] - cu[b], mq)
            if n <= seg:
                continue
            at = lib.ws_first(cu[b], b, sh, segments, T)
            mine = set(range(at, at + -(-n // seg)))
            assert min(mine) >= 0 and max(mine) < slots, (cu, b, sh, T)
            assert not order or not mine & seen, (cu, b, sh, T)
            seen |= mine
