// Integer arithmetic of the linear attention over ragged prompts that bounds its
// accesses: for kernels and host, and without HIP for a CPU build of its tests.
#pragma once

#include <stdint.h>

#ifdef __HIP__
#define EZ_HD __host__ __device__ __forceinline__
#else
#define EZ_HD inline
#endif

namespace ez {

// Rows [first, first + count) of a sequence, count <= 0 if it has none.  Offsets
// come from the device and may hold anything: both are clamped into [0, T] before
// they are subtracted, so that the difference neither wraps nor leaves the rows.
struct SeqRows {
  int first, count;
};
EZ_HD int clamp_row(int x, int T) { return x < 0 ? 0 : x > T ? T : x; }
EZ_HD SeqRows seq_rows(int begin, int end, int T, int max_q) {
  const int r = clamp_row(begin, T), n = clamp_row(end, T) - r;
  return {r, n < max_q ? n : max_q};
}

// Workspace slots (states of a kv head), one a segment, of the sequences that are cut
// into more than one.  By segment number (T / seg + B of them) or, where those are
// more, by row: the sequence at row r has the slots from floor(2 r / seg) on.  One of
// n > seg rows needs ceil(n / seg) <= floor(2 n / seg), so it ends before the slots of
// the next, and all are below floor(2 T / seg), however many sequences are not cut.
EZ_HD bool ws_by_row(int64_t segments, int64_t T, int seg_sh) { return T >> (seg_sh - 1) < segments; }
EZ_HD int64_t ws_slots(int64_t segments, int64_t T, int seg_sh) {
  return ws_by_row(segments, T, seg_sh) ? T >> (seg_sh - 1) : segments;
}
EZ_HD int ws_first(int first, int b, int seg_sh, bool by_row) {
  return by_row ? first >> (seg_sh - 1) : (first >> seg_sh) + b;
}

}  // namespace ez
