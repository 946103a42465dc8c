// Linear attention with a decay per head over packed ragged prompts, and its
// recurrent form for one token per sequence.
//
//   S_t = lambda S_{t-1} + k_t v_t^T          S [D, D] fp32 per (state slot, kv head)
//   o_t = scale * q_t^T S_t                   lambda = exp(log_decay[kv head])
//
// Query head h reads the state of kv head h / (H / Hkv).  lambda = 0 (log_decay
// -inf) is allowed: only powers lambda^n with n >= 0 appear, and lambda^0 = 1.
//
// Over prompts the work is matrix products (a chunk of 64 tokens: 2 x 64 x 128 x (64 + 128) flops a query
// head and 2 x 64 x 128 x 128 a kv head, in two or three bf16 parts).  Prompts of some thousand tokens are bound by
// latency: of the output kernel's time the matrix cores are busy for 30%, the VALU for 40%, and its two waves a SIMD
// spend a third of theirs at waits and barriers (4096 tokens of 32 / 8 heads of 128: 47 us in all, 84 MB or 1.8
// TB/s).  Longer ones come near the memory: its output kernel moves 1.09 GB at 4.1 TB/s for two prompts of 16384
// x 32 / 32 heads, but the sums have read K and V before it (411 us in all; read and written once at a copy's
// rate 219).  Single tokens are bound by the state's traffic (200 x 32 states 153 us, 845 MB: 5.5 TB/s).
//
// A sequence's state lives in a pool of slots.  A sequence whose slot lies
// outside the pool, or that an earlier sequence with tokens holds already, is
// left out whole: nothing of it is read or written, so equal slots make no race.
#include <cmath>
#include <type_traits>

#include "common.h"
#include "internal.h"
#include "prof.h"
#include "segments.h"
#include "status.h"
#include "../../include/ezops_hip.h"

namespace ez {

EZ_PROF_DEFINE(linattn)
namespace {

struct LinAttnArgs {
  const uint16_t *q, *k, *v;
  int64_t q_rs, k_rs, v_rs;   // distance of the tokens in elements
  const float* log_decay;     // [Hkv]
  float* state;               // [num_slots, Hkv, D, D] or NULL (prefill)
  const int32_t* state_slots; // [B] or NULL (slot b)
  const int32_t *cu, *past;   // prefill: [B + 1], [B] or NULL
  uint16_t* out;              // [T, H, D]
  int64_t T, num_slots, max_q;
  int seg, seg_sh;            // prefill: tokens per segment (1 << seg_sh)
  int segments;               // prefill: segment numbers
  int split;                  // prefill: blocks that share the query heads of a kv head
  float* ws;                  // prefill: [ws_slots, Hkv, D, D] or NULL (one segment a sequence)
  int ws_slots;
  bool ws_rows, ws_all;       // prefill: slots by row, not by segment number; uncut sequences have one too
  int B, H, Hkv;
  float scale;
};

// What a state keeps over n tokens, lambda^n S: where lambda^n > 1/2 as S + (lambda^n - 1) S, so that
// the factor's own rounding does not build up over many steps as that of lambda^n itself would (a
// state that is all but kept adds it up 1 / (1 - lambda^n) times); below that as the plain product,
// which the sum would cancel in.
struct Keep {
  float m;
  bool near;
};
__device__ __forceinline__ Keep keep_over(float log_decay, float n) {
  const float m = expm1f(log_decay * n);
  return m > -0.5f ? Keep{m, true} : Keep{expf(log_decay * n), false};
}
__device__ __forceinline__ Keep uniform(const Keep& k) {  // into scalar registers
  return Keep{__int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(k.m))),
              bool(__builtin_amdgcn_readfirstlane(int(k.near)))};
}
// lambda^n S + x
__device__ __forceinline__ float decayed(const Keep& k, float S, float x) {
  const float y = fmaf(k.m, S, x);
  return k.near ? S + y : y;
}

// Whether a sequence in front of b holds `slot`: one with tokens, of which a single token's call has one for every
// sequence (an idle row of a padded prompt batch may carry any slot); lengths are looked at only where a slot is
// equal.  Every thread of the block calls it (barriers inside).
template <int THREADS>
__device__ __forceinline__ bool slot_held(const LinAttnArgs& a, int b, int slot) {
  int held = 0;
  for (int c = threadIdx.x; c < b; c += THREADS) held |= a.state_slots[c] == slot;
  held = __syncthreads_or(held);
  if (!held || !a.cu) return held;
  held = 0;
  for (int c = threadIdx.x; c < b; c += THREADS)
    held |= a.state_slots[c] == slot && seq_rows(a.cu[c], a.cu[c + 1], int(a.T), int(a.max_q)).count > 0;
  return __syncthreads_or(held);
}

// Slot of sequence b, -1 if it has none: outside the pool, or held by an earlier
// sequence.  Every thread of the block calls it (barrier inside).
template <int THREADS>
__device__ __forceinline__ int slot_of(const LinAttnArgs& a, int b) {
  const int s = a.state_slots ? a.state_slots[b] : b;
  const bool held = a.state_slots && slot_held<THREADS>(a, b, s);
  return s < 0 || s >= a.num_slots || held ? -1 : s;
}

// ---- prompts: the chunked form ------------------------------------------
// A chunk of 64 tokens with state S before it, everything decayed relative to
// one of its ends, so that only powers n >= 0 appear:
//   o_i   = scale (lambda^{i+1} S^T q_i + sum_{j<=i} lambda^{i-j} (q_i . k_j) v_j)
//   S_out = lambda^n S + sum_j lambda^{n-1-j} k_j v_j^T
// A sequence is cut into segments of `seg` tokens that end at its end; only the
// first chunk of its first segment can be short, and it is filled up with zero
// tokens at its front, which leaves every power below the same for all chunks.
//
// A sequence of one segment goes through the output kernel alone (state from the pool,
// state to the pool).  Of the others the state kernel sums every segment but the last
// from zero into the workspace, the scan turns these sums into the state before
// each segment, and the output kernel starts each segment from there.  Only where the
// query heads of a kv head are shared out to several blocks (few blocks in all) does an
// uncut sequence start from a copy of its state in the workspace as well: the block that
// leaves the last state must not meet the others' reads of the first.
//
// Matrix layout (v_mfma_f32_32x32x16_bf16: lane 32h+i holds A[i][8h..8h+7] and
// B[8h..8h+7][i]; register r of lane 32h+j holds C[8(r/4)+4h+r%4][j]).  Wave w owns
// columns 32w..32w+31 of v, of the state and of the outputs:
//   P^T = K Q^T         keys x queries; its registers are the B operand of the next
//                       product as they are, if the token slots 8h..8h+7 of a 16-key
//                       step mean keys 4h..4h+3 and 8+4h..8+4h+3
//   O^T += V^T P^T      A = V^T by transposing LDS reads in that token order
//   S   += K^T (w V)    the same V registers, weighted, are the B operand; A = K^T by
//                       transposing reads whose dims come in the order that makes
//                       registers 8u..8u+7 of S dims 16u+8h..+7:
//   O^T += S^T Q^T      S's registers are the A operand with the dims in natural order,
//                       so one set of Q registers serves both products
// The three 32 x 32 blocks of P are shared out among the waves and handed round through LDS.
// fp32 operands (P, S, w V) are given to the matrix cores in bf16 parts: two for P and
// S, whose products end in one bf16 rounding (2^-16 of a term against 2^-8), three for
// w V, whose sums are the fp32 state (2^-24).
constexpr int kC = 64;  // tokens per chunk

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef int i32x2_t __attribute__((ext_vector_type(2)));

// 16-byte chunk c of row `key` of an LDS tile lies at chunk c ^ swizzle(key): the row
// reads (32 rows, one chunk) and the transposing reads (4 rows x 64 bytes per half
// wave) both spread over all banks.
template <int D>
__device__ __forceinline__ int swizzle(int key) {
  return D == 128 ? ((key & 3) << 2) | ((key >> 2) & 3) : (((key >> 1) & 1) << 2) | ((key >> 2) & 3);
}

// LDS reads as asm blocks that end in their own wait: the compiler would make an
// ordinary read wait for the next chunk's LDS DMA as well.
// All dims of 32 token rows (N = D / 16 steps), `a` = this lane's first chunk.
template <int OFF>
__device__ __forceinline__ void lds_row(uint32_t a, bf16x8_t (&r)[8]) {
  asm volatile(
      "ds_read_b128 %0, %8 offset:%16\n\tds_read_b128 %1, %9 offset:%16\n\t"
      "ds_read_b128 %2, %10 offset:%16\n\tds_read_b128 %3, %11 offset:%16\n\t"
      "ds_read_b128 %4, %12 offset:%16\n\tds_read_b128 %5, %13 offset:%16\n\t"
      "ds_read_b128 %6, %14 offset:%16\n\tds_read_b128 %7, %15 offset:%16\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
      : "v"(a), "v"(a ^ 32), "v"(a ^ 64), "v"(a ^ 96), "v"(a ^ 128), "v"(a ^ 160), "v"(a ^ 192), "v"(a ^ 224), "i"(OFF));
}
template <int OFF>
__device__ __forceinline__ void lds_row(uint32_t a, bf16x8_t (&r)[4]) {
  asm volatile(
      "ds_read_b128 %0, %4 offset:%8\n\tds_read_b128 %1, %5 offset:%8\n\t"
      "ds_read_b128 %2, %6 offset:%8\n\tds_read_b128 %3, %7 offset:%8\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
      : "v"(a), "v"(a ^ 32), "v"(a ^ 64), "v"(a ^ 96), "i"(OFF));
}
// Transposing reads (ds_read_b64_tr_b16: in each 16-lane group, lane m receives element
// m % 4 of the 8-byte rows that lanes m/4, 4 + m/4, 8 + m/4 and 12 + m/4 address): tokens
// 16s + 4h..+3 and 8 further on (row pitch P bytes) of 32 dims a tile.
// One 32-dim tile, all four 16-token steps.
template <int P>
__device__ __forceinline__ void lds_tr_steps(uint32_t a, i32x2_t (&r)[8]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%10\n\tds_read_b64_tr_b16 %1, %9 offset:%11\n\t"
      "ds_read_b64_tr_b16 %2, %8 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
      "ds_read_b64_tr_b16 %4, %8 offset:%14\n\tds_read_b64_tr_b16 %5, %9 offset:%15\n\t"
      "ds_read_b64_tr_b16 %6, %8 offset:%16\n\tds_read_b64_tr_b16 %7, %9 offset:%17\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
      : "v"(a), "v"(a ^ 32), "i"(0), "i"(8 * P), "i"(16 * P), "i"(24 * P), "i"(32 * P), "i"(40 * P), "i"(48 * P),
        "i"(56 * P));
}
// One 16-token step, all 32-dim tiles.
template <int OFF, int P>
__device__ __forceinline__ void lds_tr_tiles(uint32_t a, i32x2_t (&r)[8]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%16\n\tds_read_b64_tr_b16 %1, %9 offset:%17\n\t"
      "ds_read_b64_tr_b16 %2, %10 offset:%16\n\tds_read_b64_tr_b16 %3, %11 offset:%17\n\t"
      "ds_read_b64_tr_b16 %4, %12 offset:%16\n\tds_read_b64_tr_b16 %5, %13 offset:%17\n\t"
      "ds_read_b64_tr_b16 %6, %14 offset:%16\n\tds_read_b64_tr_b16 %7, %15 offset:%17\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
      : "v"(a), "v"(a ^ 32), "v"(a ^ 64), "v"(a ^ 96), "v"(a ^ 128), "v"(a ^ 160), "v"(a ^ 192), "v"(a ^ 224), "i"(OFF),
        "i"(OFF + 8 * P));
}
template <int OFF, int P>
__device__ __forceinline__ void lds_tr_tiles(uint32_t a, i32x2_t (&r)[4]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4 offset:%8\n\tds_read_b64_tr_b16 %1, %5 offset:%9\n\t"
      "ds_read_b64_tr_b16 %2, %6 offset:%8\n\tds_read_b64_tr_b16 %3, %7 offset:%9\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
      : "v"(a), "v"(a ^ 32), "v"(a ^ 64), "v"(a ^ 96), "i"(OFF), "i"(OFF + 8 * P));
}
// A barrier without a wait: __syncthreads() waits for outstanding LDS DMA as well, which here is the next
// chunk's.  LDS reads and writes in front of it have ended with waits of their own.
__device__ __forceinline__ void block_barrier() { asm volatile("s_barrier" ::: "memory"); }
// The same with at most N of this wave's memory operations still out.  One block, so that no store moves between the
// wait that counts it and the barrier.
template <int N>
__device__ __forceinline__ void wait_vm_barrier() {
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"(N) : "memory");
}

// Fragments of 1 KiB in a row (16 bytes a lane): twelve read, four written.
__device__ __forceinline__ void lds_frags12(uint32_t a, bf16x8_t (&r)[12]) {
  asm volatile(
      "ds_read_b128 %0, %12\n\tds_read_b128 %1, %12 offset:%13\n\tds_read_b128 %2, %12 offset:%14\n\t"
      "ds_read_b128 %3, %12 offset:%15\n\tds_read_b128 %4, %12 offset:%16\n\tds_read_b128 %5, %12 offset:%17\n\t"
      "ds_read_b128 %6, %12 offset:%18\n\tds_read_b128 %7, %12 offset:%19\n\tds_read_b128 %8, %12 offset:%20\n\t"
      "ds_read_b128 %9, %12 offset:%21\n\tds_read_b128 %10, %12 offset:%22\n\tds_read_b128 %11, %12 offset:%23\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7]),
        "=&v"(r[8]), "=&v"(r[9]), "=&v"(r[10]), "=&v"(r[11])
      : "v"(a), "i"(1 << 10), "i"(2 << 10), "i"(3 << 10), "i"(4 << 10), "i"(5 << 10), "i"(6 << 10), "i"(7 << 10),
        "i"(8 << 10), "i"(9 << 10), "i"(10 << 10), "i"(11 << 10));
}
__device__ __forceinline__ void lds_write_frags4(uint32_t a, const bf16x8_t (&r)[4]) {
  asm volatile(
      "ds_write_b128 %0, %1\n\tds_write_b128 %0, %2 offset:%5\n\tds_write_b128 %0, %3 offset:%6\n\t"
      "ds_write_b128 %0, %4 offset:%7\n\ts_waitcnt lgkmcnt(0)"
      :
      : "v"(a), "v"(r[0]), "v"(r[1]), "v"(r[2]), "v"(r[3]), "i"(1 << 10), "i"(2 << 10), "i"(3 << 10)
      : "memory");
}
// Register r: 8 (r / 4) + r % 4 floats below the address + 108.
__device__ __forceinline__ void lds_weights(uint32_t a, float (&r)[16]) {
  asm volatile(
      "ds_read_b32 %0, %16 offset:108\n\tds_read_b32 %1, %16 offset:104\n\tds_read_b32 %2, %16 offset:100\n\t"
      "ds_read_b32 %3, %16 offset:96\n\tds_read_b32 %4, %16 offset:76\n\tds_read_b32 %5, %16 offset:72\n\t"
      "ds_read_b32 %6, %16 offset:68\n\tds_read_b32 %7, %16 offset:64\n\tds_read_b32 %8, %16 offset:44\n\t"
      "ds_read_b32 %9, %16 offset:40\n\tds_read_b32 %10, %16 offset:36\n\tds_read_b32 %11, %16 offset:32\n\t"
      "ds_read_b32 %12, %16 offset:12\n\tds_read_b32 %13, %16 offset:8\n\tds_read_b32 %14, %16 offset:4\n\t"
      "ds_read_b32 %15, %16\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7]),
        "=&v"(r[8]), "=&v"(r[9]), "=&v"(r[10]), "=&v"(r[11]), "=&v"(r[12]), "=&v"(r[13]), "=&v"(r[14]), "=&v"(r[15])
      : "v"(a));
}
__device__ __forceinline__ bf16x8_t join(const i32x2_t& x, const i32x2_t& y) {
  return as_bf16x8(make_uint4(uint32_t(x[0]), uint32_t(x[1]), uint32_t(y[0]), uint32_t(y[1])));
}

// The next bf16 part of eight values: returned rounded, and taken off them.  Values that round to infinity (from 2^128
// (1 - 2^-9) on) leave NaN: the range that the entry documents ends below them.
__device__ __forceinline__ bf16x8_t take_part(float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    w[e] = cvt_bf2(x[2 * e], x[2 * e + 1]);
    x[2 * e] -= bf_lo(w[e]);
    x[2 * e + 1] -= bf_hi(w[e]);
  }
  return as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
}
__device__ __forceinline__ bf16x8_t last_part(const float (&x)[8]) {
  return as_bf16x8(make_uint4(cvt_bf2(x[0], x[1]), cvt_bf2(x[2], x[3]), cvt_bf2(x[4], x[5]), cvt_bf2(x[6], x[7])));
}

// An LDS address of this chunk's buffer.  Opaque to the compiler, which would else keep every
// address derived from it in a register of its own throughout the loop.
__device__ __forceinline__ uint32_t lds_at(uint32_t base, uint32_t off) {
  uint32_t a = base + off;
  asm volatile("" : "+v"(a));
  return a;
}

// lambda^n, n >= 0, from log2(lambda); lambda^0 = 1 for lambda = 0 too.
__device__ __forceinline__ float power(float g2, int n) { return n == 0 ? 1.f : __builtin_amdgcn_exp2f(g2 * float(n)); }

// Segment numbers: sequence b's segments are numbers cu[b] / seg + b, + 1, ...: distinct
// for distinct sequences, and at most T / seg + B in all, so the host knows the grid.
struct Segment {
  int s, count;        // index in its sequence, the sequence's number of segments
  int slot;            // state slot (-1: no pool)
  bool cont;           // the sequence starts from its stored state
  int ws;              // workspace slot of the state before the segment (-1: none)
  int row;             // first row of the segment
  int len;             // tokens
};

// Finds segment number `id`; false if there is none (every thread agrees).  Contains barriers.
template <int THREADS>
__device__ __forceinline__ bool find_segment(const LinAttnArgs& a, int id, Segment& g) {
  __shared__ int s_seq[4];
  const int T = int(a.T);
  // every thread looks at its sequences with all of their entries at once: one memory latency, not three
  int count = 0;  // sequences whose first segment number is at most id: the last of them is ours
  int begin = 0, len = 0, slot = -1, past = 0;
  for (int c0 = 0; c0 < a.B; c0 += THREADS) {
    const int c = c0 + threadIdx.x;
    bool in = false;
    if (c < a.B) {
      const SeqRows r = seq_rows(a.cu[c], a.cu[c + 1], T, int(a.max_q));
      const int sl = a.state ? (a.state_slots ? a.state_slots[c] : c) : -1, p = a.past ? a.past[c] : 0;
      in = (r.first >> a.seg_sh) + c <= id;
      if (in) begin = r.first, len = r.count, slot = sl, past = p;
    }
    count += __syncthreads_count(in);
  }
  const int b = __builtin_amdgcn_readfirstlane(count) - 1;
  if (b < 0) return false;
  if (int(threadIdx.x) == b % THREADS) {
    // offsets that do not decrease: this thread's last sequence with a number at most id is b
    s_seq[0] = begin;
    s_seq[1] = len;
    s_seq[2] = slot;
    s_seq[3] = past;
  }
  __syncthreads();
  // out of LDS into scalar registers: every thread has the same
  const int r0 = __builtin_amdgcn_readfirstlane(s_seq[0]);
  const int n = __builtin_amdgcn_readfirstlane(s_seq[1]);
  slot = __builtin_amdgcn_readfirstlane(s_seq[2]);
  past = __builtin_amdgcn_readfirstlane(s_seq[3]);
  if (a.state && (slot < 0 || slot >= a.num_slots || (a.state_slots && slot_held<THREADS>(a, b, slot)))) return false;
  const int s = id - ((r0 >> a.seg_sh) + b);
  if (n <= 0 || s < 0 || s >= (n + a.seg - 1) >> a.seg_sh) return false;
  const int cnt = (n + a.seg - 1) >> a.seg_sh;
  const int first = n - ((cnt - 1) << a.seg_sh);  // 1 .. seg
  g.s = s;
  g.count = cnt;
  g.slot = slot;
  g.cont = a.state && past > 0;
  g.ws = a.ws && (cnt > 1 || a.ws_all) ? ws_first(r0, b, a.seg_sh, a.ws_rows) + s : -1;
  g.row = r0 + (s ? first + ((s - 1) << a.seg_sh) : 0);
  g.len = s ? a.seg : first;
  return true;
}

// OUT: the outputs of a segment (and, of a sequence's last one, its last state);
// otherwise the sum of a segment from a zero state.  Block = (segment, kv head).
template <int D, bool OUT>
__global__ __launch_bounds__(2 * D) __attribute__((amdgpu_waves_per_eu(2))) void linear_attn_chunk_kernel(LinAttnArgs a) {
  EZ_PROF_WAVE(OUT ? kProfLinAttnPrefill : kProfLinAttnState);
  constexpr int THREADS = 2 * D, NT = D / 32, NK = D / 16, P = 2 * D;  // P: bytes of an LDS row
  constexpr int TILE = kC * P, LPT = TILE / 16 / THREADS;
  // K in two buffers (read up to the end of its chunk; the next one is asked for at the chunk's start), V and Q
  // in one each: asked for once the ones before are in registers.  76 KiB at D = 128: two blocks a CU.
  __shared__ __align__(1024) uint16_t Ks[2][kC * D], Vs[OUT ? 1 : 2][kC * D], Qs[OUT ? kC * D : 8];
  __shared__ __align__(1024) uint16_t Ps[OUT ? 3 * 4 * 512 : 8];  // block of P x (16-key step, part) x lane x 8
  __shared__ float pw[96];
  // The blocks that share a kv head's K, V and state are 8 apart: on one XCD, whose L2 then reads them once, and the
  // one that has summed the segment (all kernels, 4096 tokens of 32 / 8 heads: 5% less time, 1024 tokens 8%).
  const int split = OUT ? a.split : 1, units = a.segments * a.Hkv;
  const int u0 = int(blockIdx.x) / (8 * split) * 8, within = int(blockIdx.x) - u0 * split, wide = min(8, units - u0);
  const int part = within / wide, unit = u0 + within - part * wide;
  const int kvh = unit % a.Hkv, id = unit / a.Hkv;
  Segment sg;
  if (!find_segment<THREADS>(a, id, sg)) return;
  if (!OUT && sg.s == sg.count - 1) return;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, j = lane & 31;
  const int chunks = (sg.len + kC - 1) / kC, pad = chunks * kC - sg.len;
  const float g = a.log_decay[kvh];
  const float g2 = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(g * 1.4426950408889634f)));

  // state of this wave's columns: register r of tile t = S[32t + 16(r/8) + 8h + r%8][32w + j]
  f32x16_t S[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) S[t][r] = 0.f;
  const int elem = 8 * h * D + 32 * w + j;
  float* pool = sg.slot >= 0 ? a.state + (int64_t(sg.slot) * a.Hkv + kvh) * D * D : nullptr;
  float* ws = a.ws + (int64_t(max(sg.ws, 0)) * a.Hkv + kvh) * D * D;
  if (OUT && (sg.s > 0 || sg.cont)) {
    const float* src = sg.ws >= 0 ? ws : pool;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[t][r] = src[elem + (32 * t + 16 * (r >> 3) + (r & 7)) * D];
  }

  // weights of P: pw[31 + n] = scale * lambda^n, 0 for n < 0 (keys behind the query); n = query - key in the
  // blocks on the diagonal, 32 more in the one below it
  if constexpr (OUT) {
    if (tid < 96) pw[tid] = tid < 31 ? 0.f : a.scale * power(g2, tid - 31);
  }

  // staging: LDS chunk p = THREADS c + tid holds 16-byte chunk (p % (D/8)) ^ swizzle of row
  // p / (D/8).  Buffer loads: rows in front of the segment lie past the resource's end as
  // unsigned offsets and read as zeros.
  constexpr int RPL = THREADS / (D / 8);  // rows per load of the block: 16, which the swizzle does not see
  static_assert(RPL == 16 && LPT * RPL == kC, "staging covers the chunk");
  const int srow = tid / (D / 8), sch = (tid % (D / 8)) ^ swizzle<D>(srow);
  // head `hd` of chunk c's rows of x into LDS at `to`
  auto load_tile = [&](const uint16_t* x, int64_t rs, int hd, int c, uint16_t* to) {
    const int r0 = c * kC - pad;  // first row of the chunk in the segment; negative in a short first chunk
    const int rb = max(r0, 0), back = rb - r0;
    const auto res = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(x + (sg.row + rb) * rs + hd * D), 0,
                                                       int((kC - back) * 2 * rs), 0x00020000);
    const uint32_t pitch = uint32_t(2 * rs), off = uint32_t(srow) * pitch + 16 * sch;
#pragma unroll
    for (int i = 0; i < LPT; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          res, (__attribute__((address_space(3))) void*)(to + (i * THREADS + w * kWave) * 8), 16,
          off + uint32_t(i * RPL - back) * pitch, 0, 0, 0);
  };
  auto load_k = [&](int c) { load_tile(a.k, a.k_rs, kvh, c, Ks[c & 1]); };
  auto load_v = [&](int c) { load_tile(a.v, a.v_rs, kvh, c, Vs[OUT ? 0 : c & 1]); };

  // LDS read addresses in buffer 0
  const uint32_t kbase = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint16_t*)(&Ks[0][0])));
  const uint32_t vbase = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint16_t*)(&Vs[0][0])));
  const uint32_t krd = kbase + uint32_t(j * P + ((h ^ swizzle<D>(j)) << 4));
  const int mm = lane & 15, g1 = (lane >> 4) & 1, trow = 4 * h + (mm >> 2), gm = mm & 3;
  const int kg = ((gm & 1) << 1) | (gm >> 1);  // dim groups 0, 2, 1, 3
  const uint32_t ktr = kbase + uint32_t(trow * P + (((2 * g1 + (kg >> 1)) ^ swizzle<D>(trow)) << 4) + 8 * (kg & 1));
  const uint32_t vtr = vbase + uint32_t(trow * P + (((4 * w + 2 * g1 + (gm >> 1)) ^ swizzle<D>(trow)) << 4) + 8 * (gm & 1));

  const uint32_t pfr = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint16_t*)(&Ps[0]))) +
                       uint32_t(lane * 16);

  const uint32_t qrd = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint16_t*)(&Qs[0]))) +
                       uint32_t(j * P + ((h ^ swizzle<D>(j)) << 4));

  // register r wants n = j - 8 (r / 4) - 4 h - r % 4
  const uint32_t pwrd = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const float*)(&pw[0]))) +
                        uint32_t(4 * (31 + j - 4 * h - 27));
  const int G = a.H / a.Hkv / split, h0 = kvh * (a.H / a.Hkv) + part * G;  // this block's query heads
  float* dst = OUT ? (sg.s == sg.count - 1 && part == 0 ? pool : nullptr) : sg.ws + 1 < a.ws_slots ? ws + int64_t(a.Hkv) * D * D : nullptr;
  const Keep keep_first = uniform(keep_over(g, float(kC - pad))), keep_full = uniform(keep_over(g, float(kC)));
  // One 32 x 32 block of P (0: first keys and queries, 1: first keys, second queries, 2: second keys and
  // queries), weighted, in two parts: the operand of the product with V, four fragments.
  auto make_p = [&](int blk, uint32_t buf) {
    f32x16_t st;
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] = 0.f;
    {
      bf16x8_t kf[NK], qf[NK];
      lds_row<0>(lds_at(krd, buf + (blk >> 1) * 32 * P), kf);
      lds_row<0>(lds_at(qrd, (blk > 0) * 32 * P), qf);
#pragma unroll
      for (int s = 0; s < NK; ++s) st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[s], qf[s], st, 0, 0, 0);
    }
    const bool diag = blk != 1;
    float pm[16];
    lds_weights(lds_at(pwrd, diag ? 0 : 128), pm);
    bf16x8_t pf[4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int r = 8 * u + e;
        // keys behind the query give nothing, whatever they hold
        x[e] = !diag || j >= 8 * (r >> 2) + 4 * h + (r & 3) ? st[r] * pm[r] : 0.f;
      }
      pf[2 * u] = take_part(x);
      pf[2 * u + 1] = last_part(x);
    }
    lds_write_frags4(pfr + 4096 * blk, pf);
  };
  // Sums take the chunks from the last to the first, their weights counted from the segment's end: what the
  // memory-side cache still holds of K and V is then where the output kernel begins, and no sum has to be decayed
  // (all kernels, 2 x 16384 tokens of 32 / 32 heads: 4% less time, 4096 of 32 / 8 1%).
  const int c0 = OUT ? 0 : chunks - 1;
  load_k(c0);
  load_v(c0);
  if constexpr (OUT) load_tile(a.q, a.q_rs, h0, 0, Qs);
  wait_vm<0>();
  __syncthreads();
  for (int it = 0; it < chunks; ++it) {
    const int c = OUT ? it : chunks - 1 - it, cn = OUT ? c + 1 : c - 1;
    const uint32_t buf = uint32_t(c & 1) * TILE;
    const int r0 = c * kC - pad;
    const bool more = it + 1 < chunks;
    if (OUT && G == 1 && c > 0) load_v(c);  // with more heads it is asked for behind the first one
    if (more) {
      load_k(cn);
      if (!OUT) load_v(cn);
    }
    i32x2_t vf[8];
    if (!OUT) lds_tr_steps<P>(lds_at(vtr, buf), vf);
    if constexpr (OUT) {
      for (int hg = 0; hg < G; ++hg) {
        const int hq = h0 + hg;
        // blocks of P: wave w makes block w (0: first keys and queries, 1: first keys, second queries,
        // 2: second keys and queries); of two waves the first makes block 2 too
        // three blocks of P for the waves: the one that goes without (or, of two waves, the one that makes two)
        // is not on the same SIMD in the two blocks of a CU, which are 256 apart
        const int odd = (blockIdx.x >> 8) & 1, blk = D == 64 ? w : (w + 2 * odd) & 3;
        if (blk < 3) make_p(blk, buf);
        if (D == 64 && w == odd) make_p(2, buf);
        __builtin_amdgcn_sched_barrier(0);
        bf16x8_t q[2][NK];
        lds_row<0>(lds_at(qrd, 0), q[0]);
        lds_row<32 * P>(lds_at(qrd, 0), q[1]);
        __builtin_amdgcn_sched_barrier(0);
        // what the state gives, scaled by lambda^(i+1) of the query.  The parts of S are made anew for
        // every head (S is opaque here): kept, they would take the registers of S a second time.
#pragma unroll
        for (int t = 0; t < NT; ++t) asm volatile("" : "+v"(S[t]));
        f32x16_t o[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) o[0][r] = o[1][r] = 0.f;
#pragma unroll
        for (int s = 0; s < NK; ++s) {
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = S[s >> 1][8 * (s & 1) + e];
          const bf16x8_t hi = take_part(x), lo = last_part(x);
          o[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi, q[0][s], o[0], 0, 0, 0);
          o[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hi, q[1][s], o[1], 0, 0, 0);
          o[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lo, q[0][s], o[0], 0, 0, 0);
          o[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lo, q[1][s], o[1], 0, 0, 0);
        }
        // the parts of the next step between the products of this one
        __builtin_amdgcn_sched_group_barrier(0x2, 24, 0);
#pragma unroll
        for (int i = 0; i < 4 * NK; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x2, 6, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float f = a.scale * power(g2, max(r0 + 32 * t + j - max(r0, 0) + 1, 0));
#pragma unroll
          for (int r = 0; r < 16; ++r) o[t][r] *= f;
        }
        __builtin_amdgcn_sched_barrier(0);
        // P is there, Q has been read; for the first head V has landed (behind it is the next K)
        if (hg > 0 || c == 0) block_barrier();
        else if (more) wait_vm_barrier<LPT>();
        else wait_vm_barrier<0>();
        if (hg + 1 < G) load_tile(a.q, a.q_rs, hq + 1, c, Qs);
        else if (more) load_tile(a.q, a.q_rs, h0, c + 1, Qs);
        if (hg == 0) lds_tr_steps<P>(lds_at(vtr, 0), vf);
        // what the chunk's own tokens give: block 0 to the first queries, blocks 1 and 2 to the second
        bf16x8_t pa[12];
        lds_frags12(pfr, pa);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bf16x8_t v0 = join(vf[2 * (i >> 1)], vf[2 * (i >> 1) + 1]), v1 = join(vf[4 + 2 * (i >> 1)], vf[5 + 2 * (i >> 1)]);
          o[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v0, pa[4 + i], o[1], 0, 0, 0);
          o[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v0, pa[i], o[0], 0, 0, 0);
          o[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v1, pa[8 + i], o[1], 0, 0, 0);
        }
        // o[t][4e + x] = O^T[column 8e + 4h + x][query j]: the lane halves swap groups, so that each stores 16 bytes
        // of a row, columns 16p + 8h..+7.  (Through LDS to four lanes a row: 1-5% slower for its barrier.)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int row = r0 + 32 * t + j;
          uint16_t* op = a.out + (int64_t(sg.row + max(row, 0)) * a.H + hq) * D + 32 * w + 8 * h;
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const auto u = __builtin_amdgcn_permlane32_swap(cvt_bf2(o[t][8 * p], o[t][8 * p + 1]),
                                                            cvt_bf2(o[t][8 * p + 4], o[t][8 * p + 5]), false, false);
            const auto v = __builtin_amdgcn_permlane32_swap(cvt_bf2(o[t][8 * p + 2], o[t][8 * p + 3]),
                                                            cvt_bf2(o[t][8 * p + 6], o[t][8 * p + 7]), false, false);
            if (row >= 0) *reinterpret_cast<uint4*>(op + 16 * p) = make_uint4(u[0], v[0], u[1], v[1]);
          }
        }
        // The next Q has landed: behind it in the counter are this head's four stores (all there unless the
        // chunk is short).  V is in registers, P has been read.
        if (hg + 1 < G) {
          if (r0 < 0) wait_vm_barrier<0>();
          else wait_vm_barrier<4>();
          if (hg == 0 && more) load_v(c + 1);
        }
      }
    }
    if (!more && !dst) break;  // nobody takes the state on
    const Keep keep = r0 < 0 ? keep_first : keep_full;
    if (!OUT) {
      // nothing: the weights count from the segment's end
    } else if (keep.near) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[t][r] = fmaf(S[t][r], keep.m, S[t][r]);
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[t][r] *= keep.m;
    }
    // weights lambda^(15 - token) of a 16-token step, made anew for every chunk: registers are short
    float wv[8], gv = g2;
    asm volatile("" : "+v"(gv));
#pragma unroll
    for (int e = 0; e < 8; ++e) wv[e] = power(gv, 15 - (8 * (e >> 2) + 4 * h + (e & 3)));
    bf16x8_t vp[2][3];  // the parts of w V of a 16-token step, and of the one after it
    auto parts_of_v = [&](auto sc) {
      constexpr int s = decltype(sc)::value;
      float x[8];
      float f = power(g2, 48 - 16 * s + (OUT ? 0 : kC * it));
      asm volatile("" : "+v"(f));  // keeps the products f * wv out of registers of their own
      unpack8(__builtin_bit_cast(uint4, join(vf[2 * s], vf[2 * s + 1])), x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= wv[e] * f;
      vp[s & 1][0] = take_part(x);
      vp[s & 1][1] = take_part(x);
      vp[s & 1][2] = last_part(x);
    };
    auto add_step = [&](auto sc) {
      constexpr int s = decltype(sc)::value;
      i32x2_t kf[2 * NT];
      lds_tr_tiles<16 * s * P, P>(lds_at(ktr, buf), kf);
      if constexpr (s < 3) parts_of_v(std::integral_constant<int, s + 1>{});
#pragma unroll
      for (int i = 2; i >= 0; --i)  // the smallest part first
#pragma unroll
        for (int t = 0; t < NT; ++t)
          S[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(join(kf[2 * t], kf[2 * t + 1]), vp[s & 1][i], S[t], 0, 0, 0);
      // the next step's parts between this step's products
#pragma unroll
      for (int i = 0; i < 3 * NT; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, 24 / NT, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    parts_of_v(std::integral_constant<int, 0>{});
    add_step(std::integral_constant<int, 0>{});
    add_step(std::integral_constant<int, 1>{});
    add_step(std::integral_constant<int, 2>{});
    add_step(std::integral_constant<int, 3>{});
    // the next chunk (OUT: the next K and Q) has landed: behind it are at most the four stores
    if (!OUT || r0 < 0) wait_vm_barrier<0>();
    else wait_vm_barrier<4>();
  }
  if (dst) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) dst[elem + (32 * t + 16 * (r >> 3) + (r & 7)) * D] = S[t][r];
  }
}

// The workspace's slot of segment s > 0 holds the sum of segment s - 1; becomes the state
// before segment s.  Slot 0 gets the stored state where the sequence continues (the output
// kernel overwrites the pool while blocks that start from there may still have to read it);
// uncut sequences that no two blocks share have no slot and no part in this.
// Block = (sequence, kv head, 256 elements), one element a thread: the chain over the segments is
// short of work per step, so the chip is filled with threads, each eight loads ahead of its sums.
// With Hkv a multiple of 8 a kv head is on one XCD in all three kernels (workgroups go round the XCDs in turn), and
// sums and states stay in its L2 (all kernels, 32 / 8 heads: six sequences of up to 260 tokens 12% less time, 1024 tokens
// 14%, 4096 4%).
template <int D>
__global__ __launch_bounds__(256) void linear_attn_scan_kernel(LinAttnArgs a) {
  EZ_PROF_WAVE(kProfLinAttnState);
  constexpr int PARTS = D * D / 256, AHEAD = 8;
  const int kvh = blockIdx.x % a.Hkv, part = blockIdx.x / a.Hkv, b = blockIdx.y;
  const SeqRows rows = seq_rows(a.cu[b], a.cu[b + 1], int(a.T), int(a.max_q));
  const int r0 = rows.first, n = rows.count;
  if (n <= 0) return;
  const bool cont = a.state && a.past && a.past[b] > 0;
  if (n <= a.seg && !(cont && a.ws_all)) return;
  int slot = -1;
  if (a.state) {
    slot = slot_of<256>(a, b);
    if (slot < 0) return;
  }
  const int cnt = (n + a.seg - 1) >> a.seg_sh, id = ws_first(r0, b, a.seg_sh, a.ws_rows);
  const int last = min(cnt, a.ws_slots - id);  // decreasing offsets must not lead past the workspace
  const int at = part * 256 + int(threadIdx.x);
  const int64_t step = int64_t(a.Hkv) * D * D;
  float* ws = a.ws + (int64_t(id) * a.Hkv + kvh) * D * D + at;
  auto load = [&](float(&x)[AHEAD], int s0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) x[i] = ws[min(s0 + i, last - 1) * step];
  };
  float x[AHEAD], next[AHEAD];
  if (last > 1) load(x, 1);
  float S = 0.f;
  if (cont) {
    S = a.state[(int64_t(slot) * a.Hkv + kvh) * D * D + at];
    ws[0] = S;
  }
  const float g = a.log_decay[kvh];
  const Keep first = keep_over(g, float(n - ((cnt - 1) << a.seg_sh))), rest = keep_over(g, float(a.seg));
  for (int s0 = 1; s0 < last; s0 += AHEAD) {
    if (s0 + AHEAD < last) load(next, s0 + AHEAD);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (s0 + i < last) {
        S = decayed(s0 + i == 1 ? first : rest, S, x[i]);
        ws[(s0 + i) * step] = S;
      }
      x[i] = next[i];
    }
  }
}

// log2 of the tokens per segment: the longest segments that still give about 512 blocks over the whole
// batch, two a CU (2 x 16384 tokens of 32 / 32 heads, all three kernels: with 256 blocks 31% slower, with 1024 7%); two
// chunks as soon as that gives one block a CU (4096 tokens of 32 / 8: with 512 blocks of a chunk 12% slower, each segment
// costs 256 KiB of state traffic a kv head); at least a chunk.  Two chunks of one or two query heads a kv head are not
// cut at all (128 tokens of 8 / 8 heads, cut: 31% slower).  The same numbers serve heads of 64, whose blocks are half
// as many waves: with twice the blocks here and below 4096 and 16384 tokens of 32 / 8 heads take 33.5 and 86.7 us
// (31.2 and 76.2), 16384 of 32 / 32 121.7 (118.8), 300 tokens 21.6 (22.2), 64 to 1024 otherwise the same.
int segment_shift(int64_t T, int64_t G, int64_t Hkv, int64_t max_q) {
  int sh = 6;
  while ((T * Hkv) >> (sh + 1) >= (sh < 7 ? 256 : 512)) ++sh;
  return G <= 2 && max_q <= 2 * kC && sh < 7 ? 7 : sh;
}
// Blocks a kv head's query heads are shared out to where the segments alone leave CUs without work; each of them
// updates the state for itself, and the first leaves it.  Up to two a CU and 64 for the last segments of the
// sequences, which are blocks too (4096 tokens of 32 / 8 heads: 528).  64 fresh tokens of 32 / 8 heads: in one block
// a kv head 69% slower; 4096 tokens with 1056 blocks 17% slower.
int head_split(int64_t blocks, int64_t G) {
  int64_t n = 1;
  while (2 * n <= G && blocks * 2 * n <= 576) n *= 2;
  return int(n);
}
int64_t segment_count(int64_t B, int64_t T, int sh) { return (T >> sh) + B; }

// How a call is cut up: segments, blocks a kv head's query heads are shared out to, workspace slots (0: no workspace).
// Without a workspace the heads of continued states stay in one block.
struct Cut {
  int sh, split;
  int64_t segments, slots;
  bool by_row;
};
Cut cut_up(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t max_q, bool continued) {
  Cut c{};
  c.sh = segment_shift(T, H / Hkv, Hkv, max_q);
  c.segments = segment_count(B, T, c.sh);
  const bool need = max_q > int64_t(1) << c.sh;
  c.split = need || !continued ? head_split(c.segments * Hkv, H / Hkv) : 1;
  if (need) {
    // shared out heads: a slot for every sequence, at most 288 states of a kv head then (head_split)
    c.by_row = c.split == 1 && ws_by_row(c.segments, T, c.sh);
    c.slots = c.split == 1 ? ws_slots(c.segments, T, c.sh) : c.segments;
  }
  return c;
}

// One token per sequence, bound by the state's traffic, read and written once: block = (sequence, kv head), the state
// in registers between its one read and its one write.  NT: both with the non-temporal hint.
template <int D, bool NT>
__global__ __launch_bounds__(256) void linear_attn_decode_kernel(LinAttnArgs a) {
  EZ_PROF_WAVE(kProfLinAttnDecode);
  constexpr int LPR = D / 4;         // lanes per state row, 4 columns each
  constexpr int RPI = 256 / LPR;     // rows per step of the block
  constexpr int NI = D / RPI;        // rows per thread
  __shared__ float ks[D], qs[16][D];
  __shared__ float4 red[RPI][LPR];
  const int tid = threadIdx.x, c = tid % LPR, r0 = tid / LPR, G = a.H / a.Hkv;
  const int kvh = blockIdx.x % a.Hkv, b = blockIdx.x / a.Hkv;
  const int slot = slot_of<256>(a, b);
  if (slot < 0) return;
  f32x4_t* st = reinterpret_cast<f32x4_t*>(a.state + (int64_t(slot) * a.Hkv + kvh) * D * D) + c;
  f32x4_t S[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    if constexpr (NT) S[i] = __builtin_nontemporal_load(st + (r0 + i * RPI) * (D / 4));
    else S[i] = st[(r0 + i * RPI) * (D / 4)];
  }
  const Keep keep = keep_over(a.log_decay[kvh], 1.f);
  for (int i = tid; i < D; i += 256) ks[i] = bf2f(a.k[b * a.k_rs + kvh * D + i]);
  for (int i = tid; i < G * D; i += 256) qs[i / D][i % D] = bf2f(a.q[b * a.q_rs + kvh * G * D + i]) * a.scale;
  const uint2 vr = *reinterpret_cast<const uint2*>(a.v + b * a.v_rs + kvh * D + 4 * c);
  const float4 v = make_float4(bf_lo(vr.x), bf_hi(vr.x), bf_lo(vr.y), bf_hi(vr.y));
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const float kk = ks[r0 + i * RPI];
    S[i].x = decayed(keep, S[i].x, kk * v.x);
    S[i].y = decayed(keep, S[i].y, kk * v.y);
    S[i].z = decayed(keep, S[i].z, kk * v.z);
    S[i].w = decayed(keep, S[i].w, kk * v.w);
    if constexpr (NT) __builtin_nontemporal_store(S[i], st + (r0 + i * RPI) * (D / 4));
    else st[(r0 + i * RPI) * (D / 4)] = S[i];
  }
  for (int g = 0; g < G; ++g) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const float qq = qs[g][r0 + i * RPI];
      o.x += qq * S[i].x;
      o.y += qq * S[i].y;
      o.z += qq * S[i].z;
      o.w += qq * S[i].w;
    }
    __syncthreads();  // `red` of the previous head has been read
    red[r0][c] = o;
    __syncthreads();
    if (tid < D) {
      float sum = 0.f;
      for (int r = 0; r < RPI; ++r) sum += reinterpret_cast<const float*>(&red[r][0])[tid];
      a.out[(int64_t(b) * a.H + kvh * G + g) * D + tid] = f2bf(sum);
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// out [rows, H, D], the states and the workspace must not share memory with an input or each other: other blocks may
// still have to read them.
int check_out(const LinAttnArgs& a, int64_t rows, int64_t D, const char* what) {
  const int64_t states = a.num_slots * a.Hkv * D * D * 4, ws = int64_t(a.ws_slots) * a.Hkv * D * D * 4;
  bool states_meet = overlap(a.out, rows * a.H * D * 2, a.state, states);
  auto meets = [&](const uint16_t* x, int64_t rs, int64_t heads) {
    const int64_t n = ((rows - 1) * rs + heads * D) * 2;
    states_meet |= overlap(x, n, a.state, states);
    return overlap(x, n, a.out, rows * a.H * D * 2);
  };
  EZ_REQUIRE(!meets(a.q, a.q_rs, a.H) && !meets(a.k, a.k_rs, a.Hkv) && !meets(a.v, a.v_rs, a.Hkv),
             "%s: out must not overlap q, k or v", what);
  EZ_REQUIRE(!states_meet, "%s: state must not overlap q, k, v or out", what);
  const struct { const void* p; int64_t n; } in[] = {{a.log_decay, a.Hkv * 4}, {a.state_slots, a.B * int64_t(4)},
      {a.cu, (a.B + 1) * int64_t(4)}, {a.past, a.B * int64_t(4)}, {a.q, ((rows - 1) * a.q_rs + a.H * D) * 2},
      {a.k, ((rows - 1) * a.k_rs + a.Hkv * D) * 2}, {a.v, ((rows - 1) * a.v_rs + a.Hkv * D) * 2}};
  for (const auto& x : in)
    EZ_REQUIRE(!overlap(x.p, x.n, a.out, rows * a.H * D * 2) && !overlap(x.p, x.n, a.state, states) &&
                   !overlap(x.p, x.n, a.ws, ws),
               "%s: out, state or workspace overlaps an input", what);
  EZ_REQUIRE(!overlap(a.ws, ws, a.out, rows * a.H * D * 2) && !overlap(a.ws, ws, a.state, states),
             "%s: the workspace overlaps out or state", what);
  return EZ_OK;
}

int check_common(const LinAttnArgs& a, int64_t H, int64_t Hkv, int64_t D, float scale, const char* what) {
  EZ_REQUIRE(a.q && a.k && a.v && a.log_decay && a.out, "%s: null pointer", what);
  EZ_REQUIRE(Hkv >= 1 && H >= 1 && H <= 4096 && H % Hkv == 0, "%s: num_heads must be divisible by num_kv_heads", what);
  const int64_t G = H / Hkv;
  EZ_REQUIRE(G == 1 || G == 2 || G == 4 || G == 8 || G == 16, "%s: group size %d not supported (1, 2, 4, 8 or 16)", what,
             int(G));
  EZ_REQUIRE(D == 64 || D == 128, "%s: head_dim must be 64 or 128", what);
  EZ_REQUIRE(std::isfinite(scale), "%s: scale must be finite", what);
  EZ_REQUIRE(a.q_rs >= H * D && a.k_rs >= Hkv * D && a.v_rs >= Hkv * D, "%s: token strides below the heads' size", what);
  EZ_REQUIRE(a.q_rs % 8 == 0 && a.k_rs % 8 == 0 && a.v_rs % 8 == 0 && aligned16(a.q) && aligned16(a.k) &&
                 aligned16(a.v) && aligned16(a.out) && aligned16(a.state),
             "%s: q, k, v, out and state must be 16-byte aligned, token strides multiples of 8", what);
  return EZ_OK;
}

}  // namespace
}  // namespace ez

extern "C" size_t ezops_linear_attn_prefill_workspace_size(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t D,
                                                           int64_t max_q_len) {
  if (B < 1 || T < 1 || Hkv < 1 || D < 1) return 0;
  const int64_t max_q = max_q_len > 0 && max_q_len < T ? max_q_len : T;
  return size_t(ez::cut_up(B, T, H, Hkv, max_q, true).slots) * Hkv * D * D * sizeof(float);
}

extern "C" int ezops_linear_attn_prefill_bf16(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                                              const void* v, int64_t v_stride, const float* log_decay,
                                              const int32_t* cu_seqlens, const int32_t* past_lens, float* state,
                                              const int32_t* state_slots, int64_t num_slots, void* out, int64_t B,
                                              int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t max_q_len,
                                              float scale, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  ez::LinAttnArgs a{};
  a.q = static_cast<const uint16_t*>(q); a.q_rs = q_stride;
  a.k = static_cast<const uint16_t*>(k); a.k_rs = k_stride;
  a.v = static_cast<const uint16_t*>(v); a.v_rs = v_stride;
  a.log_decay = log_decay;
  a.state = state; a.state_slots = state ? state_slots : nullptr;
  a.cu = cu_seqlens; a.past = past_lens;
  a.out = static_cast<uint16_t*>(out);
  a.T = T; a.num_slots = num_slots;
  a.max_q = max_q_len > 0 && max_q_len < T ? max_q_len : T;
  const int rc = ez::check_common(a, H, Hkv, D, scale, "linear_attn_prefill");
  if (rc != EZ_OK) return rc;
  EZ_REQUIRE(cu_seqlens, "linear_attn_prefill: null pointer");
  EZ_REQUIRE(B >= 1 && B <= 65536 && T >= 1 && T < (int64_t(1) << 30),
             "linear_attn_prefill: batch must be in [1, 65536] and tokens in [1, 2^30)");
  EZ_REQUIRE(!state || (num_slots >= 1 && num_slots < (int64_t(1) << 31)),
             "linear_attn_prefill: num_slots must be in [1, 2^31)");
  EZ_REQUIRE(max_q_len >= 0, "linear_attn_prefill: max_q_len must be >= 0");
  a.B = int(B); a.H = int(H); a.Hkv = int(Hkv);
  a.scale = scale > 0.f ? scale : 1.f / sqrtf(float(D));
  EZ_REQUIRE(q_stride < (1 << 23) && k_stride < (1 << 23) && v_stride < (1 << 23),
             "linear_attn_prefill: token strides must be below 2^23");
  const ez::Cut cut = ez::cut_up(B, T, H, Hkv, a.max_q, state && past_lens);
  a.seg_sh = cut.sh;
  a.seg = 1 << a.seg_sh;
  const int64_t segments = cut.segments;
  const size_t need = size_t(cut.slots) * Hkv * D * D * sizeof(float);
  EZ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ez::aligned16(workspace)),
             "linear_attn_prefill: needs a 16-byte aligned workspace of %zu bytes", need);
  // a launch takes fewer than 2^32 threads along an axis; T / seg * Hkv is below 1024 by the rule above
  EZ_REQUIRE(segments * Hkv < (int64_t(1) << 24),
             "linear_attn_prefill: too many sequences and heads for one launch");
  a.segments = int(segments);
  a.ws = need ? static_cast<float*>(workspace) : nullptr;
  a.ws_slots = int(cut.slots);
  const int out_rc = ez::check_out(a, T, D, "linear_attn_prefill");
  if (out_rc != EZ_OK) return out_rc;
  a.ws_rows = cut.by_row;
  a.ws_all = cut.split > 1;
  a.split = cut.split;
  const dim3 grid(unsigned(segments * Hkv)), outs(unsigned(segments * Hkv * a.split)), parts(unsigned(Hkv * (D * D / 256)), unsigned(B));
  if (D == 64) {
    if (need) {
      hipLaunchKernelGGL((ez::linear_attn_chunk_kernel<64, false>), grid, dim3(128), 0, stream, a);
      hipLaunchKernelGGL(ez::linear_attn_scan_kernel<64>, parts, dim3(256), 0, stream, a);
    }
    hipLaunchKernelGGL((ez::linear_attn_chunk_kernel<64, true>), outs, dim3(128), 0, stream, a);
  } else {
    if (need) {
      hipLaunchKernelGGL((ez::linear_attn_chunk_kernel<128, false>), grid, dim3(256), 0, stream, a);
      hipLaunchKernelGGL(ez::linear_attn_scan_kernel<128>, parts, dim3(256), 0, stream, a);
    }
    hipLaunchKernelGGL((ez::linear_attn_chunk_kernel<128, true>), outs, dim3(256), 0, stream, a);
  }
  return ez::launch_status("linear_attn_prefill");
}

extern "C" int ezops_linear_attn_decode_bf16(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                                             const void* v, int64_t v_stride, const float* log_decay, float* state,
                                             const int32_t* state_slots, int64_t num_slots, void* out, int64_t B,
                                             int64_t H, int64_t Hkv, int64_t D, float scale, hipStream_t stream) {
  ez::LinAttnArgs a{};
  a.q = static_cast<const uint16_t*>(q); a.q_rs = q_stride;
  a.k = static_cast<const uint16_t*>(k); a.k_rs = k_stride;
  a.v = static_cast<const uint16_t*>(v); a.v_rs = v_stride;
  a.log_decay = log_decay;
  a.state = state; a.state_slots = state_slots;
  a.out = static_cast<uint16_t*>(out);
  a.num_slots = num_slots;
  const int rc = ez::check_common(a, H, Hkv, D, scale, "linear_attn_decode");
  if (rc != EZ_OK) return rc;
  EZ_REQUIRE(state, "linear_attn_decode: null pointer");
  EZ_REQUIRE(B >= 1 && B <= 65536, "linear_attn_decode: batch must be in [1, 65536]");
  EZ_REQUIRE(num_slots >= 1 && num_slots < (int64_t(1) << 31), "linear_attn_decode: num_slots must be in [1, 2^31)");
  EZ_REQUIRE(B * Hkv < (int64_t(1) << 24),  // a launch takes fewer than 2^32 threads along an axis
             "linear_attn_decode: too many sequences and heads for one launch");
  a.B = int(B); a.H = int(H); a.Hkv = int(Hkv);
  a.scale = scale > 0.f ? scale : 1.f / sqrtf(float(D));
  const int out_rc = ez::check_out(a, B, D, "linear_attn_decode");
  if (out_rc != EZ_OK) return out_rc;
  const dim3 grid(unsigned(B * Hkv));
  // With the hint from 4 MB of states on: a step comes back to them after all other layers, from outside the caches
  // (32 heads of 128, 2 / 8 / 32 / 128 / 400 MB: 4.8 / 7.4 / 17.3 / 53.8 / 169 us without, 5.1 / 5.8 / 12.7 / 51.1 / 155
  // with it).  Only a layer alone, whose states the memory-side cache holds from step to step, is faster without it
  // (128 MB 41 and 49 us, but 32 MB 10.6 and 9.9).
  const bool nt = B * Hkv * D * D * 4 >= int64_t(4) << 20;
  if (D == 64) {
    if (nt) hipLaunchKernelGGL((ez::linear_attn_decode_kernel<64, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((ez::linear_attn_decode_kernel<64, false>), grid, dim3(256), 0, stream, a);
  } else {
    if (nt) hipLaunchKernelGGL((ez::linear_attn_decode_kernel<128, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((ez::linear_attn_decode_kernel<128, false>), grid, dim3(256), 0, stream, a);
  }
  return ez::launch_status("linear_attn_decode");
}
