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

}  // namespace ez
