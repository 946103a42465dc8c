// Per-head QK RMSNorm + rotary positions with several axes + cache write by
// slot, for packed tokens (a prompt of text and images, or one token each of
// many sequences).
//
//   y = x * rsqrt(mean(x^2) + eps) * w                 (norm optional)
//   o_i = y_i cos - y_{i+D/2} sin,  o_{i+D/2} = y_{i+D/2} cos + y_i sin
//   cos, sin = table[pos[axis(i)][t]][i],  i < D/2
//
// in fp32 with one bf16 rounding; products and sums by the explicit
// round-to-nearest intrinsics, so no contraction changes the rounding.  Pair i
// belongs to the axis in whose section it falls, or with interleaved sections to
// axis i % A while that axis has pairs left, else to axis 0.
//
// The work is memory traffic: q and k in and out, v into the cache, 2 D bytes a
// head each; the table rows are shared by the heads of a token.
#include "common.h"
#include "internal.h"
#include "prof.h"
#include "status.h"
#include "../../include/ezops_hip.h"

namespace ez {

EZ_PROF_DEFINE(mrope)
namespace {

constexpr int kMaxAxes = 4;
constexpr int kMropeMaxPairs = 4;  // pairs per lane of the scalar kernel: D <= 512

struct MropeArgs {
  const uint16_t *q, *k, *v;
  int64_t q_rs, k_rs, v_rs;  // distance of the tokens in elements
  const uint16_t *qw, *kw;   // NULL = unit weights
  const void *cos, *sin;     // [S, D], bf16 or fp32; the first D/2 columns are read
  const int32_t* positions;  // [A, T]
  const int64_t* slots;      // [T]
  uint16_t *Kc, *Vc;         // [num_pages, Hkv, page_size, D] or NULL
  uint16_t *q_out, *k_out;   // [T, H, D], [T, Hkv, D] (k_out may be NULL with a cache)
  int64_t T, S, num_slots;
  int H, Hkv, D, A, interleaved, norm, page_sh, table_f32;
  int sec[kMaxAxes];
  float eps;
};

__device__ __forceinline__ int axis_of(const MropeArgs& a, int i) {
  if (a.interleaved) {
    const int r = i % a.A;
    return i < a.A * a.sec[r] ? r : 0;
  }
  int end = a.sec[0], ax = 0;
#pragma unroll
  for (int n = 1; n < kMaxAxes; ++n) {
    ax += i >= end;
    end += a.sec[n];
  }
  return ax;
}

__device__ __forceinline__ float table_at(const MropeArgs& a, const void* t, int64_t i) {
  return a.table_f32 ? static_cast<const float*>(t)[i] : bf2f(static_cast<const uint16_t*>(t)[i]);
}

// Element offset of cache slot `s`, kv head `h`.
__device__ __forceinline__ int64_t slot_offset(const MropeArgs& a, int64_t s, int h) {
  const int64_t page = s >> a.page_sh, row = s - (page << a.page_sh);
  return (((page * a.Hkv + h) << a.page_sh) + row) * a.D;
}

// One wave per (token, head): lane l owns the pairs l, l + 64, ...; any even D
// and any alignment.
__global__ __launch_bounds__(256) void qk_norm_mrope_kernel(MropeArgs a) {
  EZ_PROF_WAVE(kProfQkMrope);
  const int lane = threadIdx.x & (kWave - 1);
  const int heads = a.H + a.Hkv;
  const int64_t units = a.T * heads;
  for (int64_t u = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); u < units; u += int64_t(gridDim.x) * 4) {
    const int64_t t = u / heads;
    const int h = int(u - t * heads);
    const bool is_q = h < a.H;
    const int kvh = h - a.H;
    int64_t pos[kMaxAxes];
    bool ok = true;
#pragma unroll
    for (int n = 0; n < kMaxAxes; ++n) {
      pos[n] = n < a.A ? int64_t(a.positions[n * a.T + t]) : 0;
      ok &= pos[n] >= 0 && pos[n] < a.S;
    }
    if (!ok) continue;
    const uint16_t* src = is_q ? a.q + t * a.q_rs + int64_t(h) * a.D : a.k + t * a.k_rs + int64_t(kvh) * a.D;
    const uint16_t* w = is_q ? a.qw : a.kw;
    const int half = a.D / 2;
    float x1[kMropeMaxPairs], x2[kMropeMaxPairs], ss = 0.f;
#pragma unroll
    for (int n = 0; n < kMropeMaxPairs; ++n) {
      const int i = lane + n * kWave;
      x1[n] = i < half ? bf2f(src[i]) : 0.f;
      x2[n] = i < half ? bf2f(src[i + half]) : 0.f;
      ss += x1[n] * x1[n] + x2[n] * x2[n];
    }
    const float r = a.norm ? rsqrtf(wave_sum(ss) / float(a.D) + a.eps) : 1.f;
    const int64_t slot = !is_q && a.Kc ? a.slots[t] : -1;
    const bool cached = slot >= 0 && slot < a.num_slots;
    uint16_t* dst = is_q ? a.q_out + (t * a.H + h) * a.D : a.k_out ? a.k_out + (t * a.Hkv + kvh) * a.D : nullptr;
    const int64_t coff = cached ? slot_offset(a, slot, kvh) : 0;
#pragma unroll
    for (int n = 0; n < kMropeMaxPairs; ++n) {
      const int i = lane + n * kWave;
      if (i >= half) break;
      float y1 = x1[n], y2 = x2[n];
      if (a.norm) {
        y1 = __fmul_rn(y1, r);
        y2 = __fmul_rn(y2, r);
        if (w) {
          y1 = __fmul_rn(y1, bf2f(w[i]));
          y2 = __fmul_rn(y2, bf2f(w[i + half]));
        }
      }
      const int ax = axis_of(a, i);
      const int64_t p = ax == 0 ? pos[0] : ax == 1 ? pos[1] : ax == 2 ? pos[2] : pos[3];
      const float c = table_at(a, a.cos, p * a.D + i), s = table_at(a, a.sin, p * a.D + i);
      const uint16_t b1 = f2bf(__fadd_rn(__fmul_rn(y1, c), __fmul_rn(-y2, s)));
      const uint16_t b2 = f2bf(__fadd_rn(__fmul_rn(y2, c), __fmul_rn(y1, s)));
      if (dst) {
        dst[i] = b1;
        dst[i + half] = b2;
      }
      if (cached) {
        a.Kc[coff + i] = b1;
        a.Kc[coff + i + half] = b2;
      }
    }
    if (cached) {
      const uint16_t* vs = a.v + t * a.v_rs + int64_t(kvh) * a.D;
      for (int i = lane; i < a.D; i += kWave) a.Vc[coff + i] = vs[i];
    }
  }
}

int launch_mrope(const MropeArgs& a, hipStream_t s) {
  const int64_t blocks = (a.T * (a.H + a.Hkv) + 3) / 4;
  hipLaunchKernelGGL(qk_norm_mrope_kernel, dim3(unsigned(blocks < (1 << 20) ? blocks : 1 << 20)), dim3(256), 0, s, a);
  return launch_status("qk_norm_mrope");
}

}  // namespace
}  // namespace ez

extern "C" int ezops_qk_norm_mrope_bf16(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                        int64_t v_stride, const void* q_norm_w, const void* k_norm_w, int norm,
                                        const void* cos, const void* sin, int table_f32, const int32_t* positions,
                                        int64_t axes, const int64_t* sections, int interleaved,
                                        const int64_t* slot_mapping, void* K_cache, void* V_cache, int64_t num_pages,
                                        int64_t page_size, void* q_out, void* k_out, int64_t T, int64_t H, int64_t Hkv,
                                        int64_t D, int64_t S, float eps, hipStream_t stream) {
  EZ_REQUIRE(q && k && cos && sin && positions && sections && q_out, "qk_norm_mrope: null pointer");
  EZ_REQUIRE(T >= 1 && T < (int64_t(1) << 30) && S >= 1 && S < (int64_t(1) << 31),
             "qk_norm_mrope: tokens must be in [1, 2^30) and table rows in [1, 2^31)");
  EZ_REQUIRE(H >= 1 && Hkv >= 1 && H <= 4096 && H % Hkv == 0,
             "qk_norm_mrope: num_heads must be in [1, 4096] and divisible by num_kv_heads");
  EZ_REQUIRE(D >= 2 && D <= 2 * ez::kMropeMaxPairs * ez::kWave && D % 2 == 0,
             "qk_norm_mrope: head_dim must be even and <= %d", 2 * ez::kMropeMaxPairs * ez::kWave);
  EZ_REQUIRE(q_stride >= H * D && k_stride >= Hkv * D && (!v || v_stride >= Hkv * D),
             "qk_norm_mrope: token strides below the heads' size");
  EZ_REQUIRE(axes >= 1 && axes <= ez::kMaxAxes, "qk_norm_mrope: 1 to %d position axes", ez::kMaxAxes);
  ez::MropeArgs a{};
  int64_t sum = 0;
  for (int64_t n = 0; n < axes; ++n) {
    EZ_REQUIRE(sections[n] >= 0 && sections[n] <= D / 2, "qk_norm_mrope: sections must be in [0, head_dim / 2]");
    EZ_REQUIRE(!interleaved || n == 0 || sections[n] == 0 || axes * (sections[n] - 1) + n < D / 2,
               "qk_norm_mrope: an interleaved section has more pairs than turns");
    sum += sections[n];
    a.sec[n] = int(sections[n]);
  }
  EZ_REQUIRE(sum == D / 2, "qk_norm_mrope: sections must add up to head_dim / 2");
  EZ_REQUIRE((K_cache == nullptr) == (V_cache == nullptr), "qk_norm_mrope: K_cache and V_cache go together");
  EZ_REQUIRE(!K_cache || (v && slot_mapping), "qk_norm_mrope: a cache needs v and slot_mapping");
  EZ_REQUIRE(!K_cache || (page_size >= 32 && page_size <= (1 << 20) && (page_size & (page_size - 1)) == 0 &&
                          num_pages >= 1 && num_pages < (int64_t(1) << 31)),
             "qk_norm_mrope: page_size must be a power of two in [32, 2^20] and num_pages in [1, 2^31)");
  EZ_REQUIRE(K_cache || k_out, "qk_norm_mrope: k needs a cache or k_out");
  a.q = static_cast<const uint16_t*>(q); a.q_rs = q_stride;
  a.k = static_cast<const uint16_t*>(k); a.k_rs = k_stride;
  a.v = static_cast<const uint16_t*>(v); a.v_rs = v_stride;
  a.qw = static_cast<const uint16_t*>(q_norm_w); a.kw = static_cast<const uint16_t*>(k_norm_w);
  a.cos = cos; a.sin = sin; a.table_f32 = table_f32 != 0;
  a.positions = positions; a.slots = slot_mapping;
  a.Kc = static_cast<uint16_t*>(K_cache); a.Vc = static_cast<uint16_t*>(V_cache);
  a.q_out = static_cast<uint16_t*>(q_out); a.k_out = static_cast<uint16_t*>(k_out);
  a.T = T; a.S = S; a.H = int(H); a.Hkv = int(Hkv); a.D = int(D); a.A = int(axes);
  a.interleaved = interleaved != 0; a.norm = norm != 0; a.eps = eps;
  if (K_cache) {
    a.page_sh = __builtin_ctzll(static_cast<unsigned long long>(page_size));
    a.num_slots = num_pages * page_size;
  }
  return ez::launch_mrope(a, stream);
}
