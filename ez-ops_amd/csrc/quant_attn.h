// Arguments and checks that the kernels of attention over the 8-bit cache share.
#pragma once

#include <array>

#include "common.h"
#include "kv8.h"

namespace ez {

struct QuantAttnArgs {
  Kv8Args c;
  const uint16_t* q;        // [T, H, D], tokens q_rs elements apart
  int64_t q_rs;
  uint16_t* out;            // [T, H, D]
  const int32_t* table;     // [B, M]
  const int32_t* kv_lens;   // decode: [B]
  const int32_t *cu, *past;  // prefill: [B + 1], [B] or NULL
  int64_t B, T, M, cap;     // cap: rows of a sequence that are read at most
  int H;
  float scale;
};

inline bool kv8_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr float kLog2e = 1.4426950408889634f;
// Factor of the scores of a block with exponent e, scale log2(e) 2^(e - 127): NaN for 255, else
// kept within (0, FLT_MAX], so that a masked score of -inf stays one and a score of 0 too
// (0 * -inf and inf * 0 are NaN).  Where it is subnormal it is off by less than 2^-148, and
// times a sum q . codes of less than 2^128 by less than 2^-20.  Callers keep it below 2^128
// where a row is not all zeros.
__device__ __forceinline__ float kv8_factor(float scale, int e) {  // e as kv8_exp gives it
  // the power first: exact where the scale is subnormal and it is large
  const float c = scale * __uint_as_float(uint32_t(e) << 23) * kLog2e;
  return e == kKvNanExp ? __uint_as_float(0x7fc00000u) : __builtin_amdgcn_fmed3f(c, 0x1p-149f, 0x1.fffffep127f);
}

constexpr float kLowest = -3e38f;  // softmax reference before any row: finite, so that differences are

// Joins n partials of a query row: (m, l) ml_step apart, 4 dims of O o_step apart, kPer of
// each in flight.  out = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s.
template <int kPer>
__device__ __forceinline__ void join_parts(const float2* ml, const float4* po, int64_t ml_step, int64_t o_step, int n,
                                           float (&out)[4]) {
  float m = kLowest, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < n; s0 += kPer) {
    float2 x[kPer];
    float4 p[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int s = min(s0 + i, n - 1);
      x[i] = ml[s * ml_step];
      p[i] = po[s * o_step];
    }
    float mn = m;
#pragma unroll
    for (int i = 0; i < kPer; ++i) mn = fmaxf(mn, x[i].x);
    const float back = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= back;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] *= back;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float f = s0 + i < n ? __builtin_amdgcn_exp2f(x[i].x - m) : 0.f;  // behind the last: the last again
      l = fmaf(f, x[i].y, l);
      o[0] = fmaf(f, p[i].x, o[0]);
      o[1] = fmaf(f, p[i].y, o[1]);
      o[2] = fmaf(f, p[i].z, o[2]);
      o[3] = fmaf(f, p[i].w, o[3]);
    }
  }
  const float inv = 1.f / l;
#pragma unroll
  for (int k = 0; k < 4; ++k) out[k] = o[k] * inv;
}

struct Range {
  const void* p;
  int64_t n;
};
// Memory of the call's tensors: out, then the inputs.
inline std::array<Range, 10> attn8_tensors(const QuantAttnArgs& a, int64_t H) {
  const int64_t pool = kv8_pool_bytes(a.c), sc = kv8_scale_bytes(a.c), row = H * a.c.D;
  return {{{a.out, a.T * row * 2}, {a.c.K, pool}, {a.c.V, pool}, {a.c.Ks, sc}, {a.c.Vs, sc}, {a.table, a.B * a.M * 4},
           {a.kv_lens, a.B * 4}, {a.cu, (a.B + 1) * 4}, {a.past, a.B * 4}, {a.q, ((a.T - 1) * a.q_rs + row) * 2}}};
}

// H, Hkv and D as the caller gave them: those in `a` are 32 bits of them.
inline int check_attn8(const char* op, const QuantAttnArgs& a, int64_t page_size, int64_t block, int64_t H, int64_t Hkv,
                       int64_t D, int64_t max_kv_len) {
  EZ_REQUIRE(a.q && a.out && a.table, "%s: null pointer", op);
  EZ_REQUIRE(D == 64 || D == 128, "%s: head_dim must be 64 or 128", op);
  EZ_REQUIRE(H >= 1 && Hkv >= 1 && H <= 4096 && H % Hkv == 0,
             "%s: num_heads must be in [1, 4096] and divisible by num_kv_heads", op);
  const int rc = check_kv8(op, a.c, page_size, block);
  if (rc != EZ_OK) return rc;
  EZ_REQUIRE(a.B >= 1 && a.B <= 65536, "%s: batch must be in [1, 65536]", op);
  EZ_REQUIRE(a.T >= 1 && a.T < (int64_t(1) << 30), "%s: tokens must be in [1, 2^30)", op);
  const int64_t G = H / Hkv;
  EZ_REQUIRE(G == 1 || G == 2 || G == 4 || G == 8 || G == 16, "%s: group size must be 1, 2, 4, 8 or 16", op);
  EZ_REQUIRE(a.M >= 1 && a.M * page_size <= (int64_t(1) << 30),
             "%s: max_pages must be >= 1 and max_pages * page_size at most 2^30", op);
  EZ_REQUIRE(max_kv_len >= 0, "%s: max_kv_len must be >= 0", op);
  EZ_REQUIRE(a.q_rs >= H * a.c.D, "%s: token strides below the heads' size", op);
  EZ_REQUIRE(a.q_rs % 8 == 0 && kv8_aligned16(a.q) && kv8_aligned16(a.out), "%s: rows of q and out must begin at multiples of 16 bytes",
             op);
  EZ_REQUIRE(a.scale < INFINITY, "%s: scale must be finite", op);
  const auto in = attn8_tensors(a, H);
  for (size_t i = 1; i < in.size(); ++i)
    EZ_REQUIRE(!overlap(a.out, in[0].n, in[i].p, in[i].n), "%s: out overlaps an input", op);
  return EZ_OK;
}

inline void finish_args(QuantAttnArgs& a, int64_t page_size, int64_t max_kv_len) {
  a.cap = a.M * page_size;
  if (max_kv_len > 0 && max_kv_len < a.cap) a.cap = max_kv_len;
  if (!(a.scale > 0.f)) a.scale = 1.f / sqrtf(float(a.c.D));
}

}  // namespace ez
