// Batch plan: from the request lengths of a ragged batch to what its kernels
// take, on the GPU: row offsets, cache lengths, positions, cache slots and the
// block table with the pages that the new tokens need.
//
//   n_b    = cu[b+1] - cu[b],  cu[b] = min(sum of the new tokens before b, T)
//   kv_b   = min(past_b + n_b, M P)                  (P rows a page, M pages a sequence)
//   have_b = ceil(past_b / P),  need_b = ceil(kv_b / P)
//   page j of b in [have_b, need_b) has rank  sum_{c<b} (need_c - have_c) + j - have_b
//   among the new pages and takes free_pages[head + rank].
//   row t of b sits at position p = past_b + t - cu[b], slot page(b, p / P) P + p % P.
//
// One launch and no hand-off between blocks: every block scans the lengths
// itself (B <= 4096 values from the L2, two block scans in LDS) and then serves
// its own rows, one per thread.  A new page begins at a row that is new itself,
// so the thread of that row enters it into the table; entries below have_b
// are only read, entries from have_b on only written, so no two threads meet.
// Latency is all it is: 3.5 us for 64 sequences of a token, 5.9 us for 512 with
// 32768 rows (a launch, the lengths, the scans, a table or list entry, the stores).
#include "common.h"
#include "internal.h"
#include "prof.h"
#include "status.h"
#include "../../include/ezops_hip.h"

namespace ez {

EZ_PROF_DEFINE(batchplan)
namespace {

constexpr int kPlanThreads = 256;
constexpr int64_t kPlanMaxBatch = 4096;  // 8 bytes of LDS per sequence

struct PlanArgs {
  const int32_t *q_lens, *past_lens;
  int32_t* table;
  const int32_t *free_pages, *span;
  int32_t *cu, *kv, *positions;
  int64_t* slots;
  int32_t* span_out;
  int64_t T, M, NP, NF;
  int B, sh;  // page_size = 1 << sh
};

// Exclusive sum over the block's threads of one value each; `total` is the sum
// over all of them.  `red` holds a value per wave.
__device__ __forceinline__ int64_t block_exclusive(int64_t v, int64_t* red, int64_t& total) {
  const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
  int64_t inc = v;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int64_t u = __shfl_up(inc, o, kWave);
    if (lane >= o) inc += u;
  }
  __syncthreads();  // `red` of a previous scan has been read
  if (lane == kWave - 1) red[w] = inc;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kPlanThreads / kWave; ++i) {
    if (i < w) before += red[i];
    total += red[i];
  }
  return before + inc - v;
}

__global__ __launch_bounds__(kPlanThreads) void batch_plan_kernel(PlanArgs a) {
  EZ_PROF_WAVE(kProfBatchPlan);
  extern __shared__ int32_t lds[];
  int32_t* cu = lds;             // [B + 1]
  int32_t* first = lds + a.B + 1;  // [B] rank of the sequence's first new page
  __shared__ int64_t red[kPlanThreads / kWave];
  const int tid = threadIdx.x, B = a.B;
  const int64_t cap = a.M << a.sh;
  const int64_t head = a.span[0];
  const int64_t tail = min(int64_t(a.span[1]), a.NF);
  const int per = (B + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per, B), b1 = min(b0 + per, B);

  int64_t sum = 0, total;
  for (int b = b0; b < b1; ++b) sum += max(a.q_lens[b], 0);
  int64_t run = block_exclusive(sum, red, total);
  for (int b = b0; b < b1; ++b) {
    cu[b] = int32_t(min(run, a.T));
    run += max(a.q_lens[b], 0);
  }
  const int64_t rows = min(total, a.T);
  if (tid == 0) cu[B] = int32_t(rows);
  __syncthreads();

  auto past_of = [&](int b) { return min(a.past_lens ? int64_t(max(a.past_lens[b], 0)) : int64_t(0), cap); };
  auto pages = [&](int64_t n) { return (n + (int64_t(1) << a.sh) - 1) >> a.sh; };
  sum = 0;
  for (int b = b0; b < b1; ++b) {
    const int64_t past = past_of(b), kv = min(past + cu[b + 1] - cu[b], cap);
    sum += pages(kv) - pages(past);
    if (blockIdx.x == 0) {
      a.cu[b] = cu[b];
      a.kv[b] = int32_t(kv);
    }
  }
  int64_t needed;
  run = block_exclusive(sum, red, needed);
  for (int b = b0; b < b1; ++b) {
    first[b] = int32_t(run);
    const int64_t past = past_of(b), kv = min(past + cu[b + 1] - cu[b], cap);
    run += pages(kv) - pages(past);
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.cu[B] = int32_t(rows);
    const int64_t avail = head < 0 ? 0 : max(tail - head, int64_t(0));
    a.span_out[0] = int32_t(head + min(needed, avail));
    a.span_out[1] = a.span[1];
    a.span_out[2] = int32_t(needed);
  }
  __syncthreads();

  for (int64_t t = int64_t(blockIdx.x) * kPlanThreads + tid; t < a.T; t += int64_t(gridDim.x) * kPlanThreads) {
    int64_t pos = -1, slot = -1;
    if (t < rows) {
      int lo = 0, hi = B - 1;  // the last sequence that begins at or before t: empty ones begin where the next does
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= t) lo = mid; else hi = mid - 1;
      }
      const int b = lo;
      const int64_t past = past_of(b);
      pos = past + t - cu[b];
      if (pos < cap) {
        const int64_t j = pos >> a.sh, have = pages(past);
        const int64_t off = pos - (j << a.sh);
        int64_t id;
        if (j < have) {
          id = a.table[b * a.M + j];
        } else {
          const int64_t at = head + first[b] + j - have;
          id = head >= 0 && at < tail ? a.free_pages[at] : -1;
        }
        if (id < 0 || id >= a.NP) id = -1;
        if (j >= have && off == 0) a.table[b * a.M + j] = int32_t(id);
        if (id >= 0) slot = (id << a.sh) + off;
      }
    }
    a.positions[t] = int32_t(pos);
    a.slots[t] = slot;
  }
}

}  // namespace
}  // namespace ez

extern "C" int ezops_paged_batch_plan(const int32_t* q_lens, const int32_t* past_lens, int32_t* block_table,
                                      const int32_t* free_pages, const int32_t* free_span, int32_t* cu_seqlens,
                                      int32_t* kv_lens, int32_t* positions, int64_t* slot_mapping,
                                      int32_t* free_span_out, int64_t B, int64_t T, int64_t page_size,
                                      int64_t max_pages, int64_t num_pages, int64_t num_free, hipStream_t stream) {
  EZ_REQUIRE(q_lens && block_table && free_span && cu_seqlens && kv_lens && positions && slot_mapping && free_span_out,
             "paged_batch_plan: null pointer");
  EZ_REQUIRE(free_pages || num_free == 0, "paged_batch_plan: null free_pages");
  EZ_REQUIRE(free_span != free_span_out, "paged_batch_plan: free_span_out must not be free_span");
  EZ_REQUIRE(B >= 1 && B <= ez::kPlanMaxBatch, "paged_batch_plan: batch must be in [1, %d]", int(ez::kPlanMaxBatch));
  EZ_REQUIRE(T >= 1 && T < (int64_t(1) << 30), "paged_batch_plan: rows must be in [1, 2^30)");
  EZ_REQUIRE(page_size >= 32 && page_size <= (1 << 20) && (page_size & (page_size - 1)) == 0,
             "paged_batch_plan: page_size must be a power of two in [32, 2^20]");
  EZ_REQUIRE(max_pages >= 1 && max_pages <= (int64_t(1) << 30) / page_size,
             "paged_batch_plan: max_pages * page_size must be in [page_size, 2^30]");
  EZ_REQUIRE(num_pages >= 1 && num_pages < (int64_t(1) << 31) && num_free >= 0 && num_free < (int64_t(1) << 30),
             "paged_batch_plan: num_pages must be in [1, 2^31) and num_free in [0, 2^30)");
  // every block reads the inputs for itself, the first while others still have to: no output may be one of them
  const struct { const void* p; int64_t n; } in[] = {{q_lens, 4 * B}, {past_lens, 4 * B}, {free_pages, 4 * num_free}, {free_span, 8}},
      out[] = {{cu_seqlens, 4 * (B + 1)}, {kv_lens, 4 * B}, {positions, 4 * T}, {slot_mapping, 8 * T}, {free_span_out, 12},
               {block_table, 4 * B * max_pages}};
  for (const auto& x : in)
    for (const auto& y : out)
      EZ_REQUIRE(!ez::overlap(x.p, x.n, y.p, y.n), "paged_batch_plan: an output overlaps an input (copy the lengths or the "
                 "span of the plan before that is written again)");
  for (const auto& x : out)
    for (const auto& y : out)
      EZ_REQUIRE(&x == &y || !ez::overlap(x.p, x.n, y.p, y.n), "paged_batch_plan: two outputs overlap");
  ez::PlanArgs a{};
  a.q_lens = q_lens; a.past_lens = past_lens;
  a.table = block_table;
  a.free_pages = free_pages; a.span = free_span;
  a.cu = cu_seqlens; a.kv = kv_lens; a.positions = positions; a.slots = slot_mapping; a.span_out = free_span_out;
  a.T = T; a.M = max_pages; a.NP = num_pages; a.NF = num_free;
  a.B = int(B);
  a.sh = __builtin_ctzll(static_cast<unsigned long long>(page_size));
  const int64_t tiles = (T + ez::kPlanThreads - 1) / ez::kPlanThreads;
  const unsigned blocks = unsigned(tiles < 1024 ? tiles : 1024);
  hipLaunchKernelGGL(ez::batch_plan_kernel, dim3(blocks), dim3(ez::kPlanThreads), size_t(2 * B + 1) * sizeof(int32_t),
                     stream, a);
  return ez::launch_status("paged_batch_plan");
}
