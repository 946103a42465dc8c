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
// head each; the table rows are shared by the heads of a token.  Measured: 16384
// tokens of 32 + 2 x 8 heads of 128 78 us, 5.2 TB/s (a large copy reaches 4.9); 4097
// tokens of 16 + 2 x 8 14.4 us; 16 tokens 5.3 us, a launch and three dependent loads.
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

// Sum over the LPG lanes of a group (4, 8, 16 or 32 neighbours); every lane gets it.
template <int LPG>
__device__ __forceinline__ float group_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xF, 0xF, true));   // quad_perm [1,0,3,2]
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xF, 0xF, true));   // quad_perm [2,3,0,1]
  if constexpr (LPG >= 8)
    v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xF, 0xF, true));  // row_half_mirror
  if constexpr (LPG >= 16)
    v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x140, 0xF, 0xF, true));  // row_mirror
  if constexpr (LPG >= 32) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  return v;
}

// Table entries of this lane's 8 pairs at row p.
__device__ __forceinline__ void load8(const uint16_t* p, float (&f)[8]) { unpack8(*reinterpret_cast<const uint4*>(p), f); }
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 x = reinterpret_cast<const float4*>(p)[0], y = reinterpret_cast<const float4*>(p)[1];
  f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w;
  f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
}

// 16-byte accesses, with the non-temporal hint where NT.
template <bool NT>
__device__ __forceinline__ uint4 load16(const uint16_t* p) {
  if constexpr (NT) return ld16_stream(p);
  return *reinterpret_cast<const uint4*>(p);
}
template <bool NT>
__device__ __forceinline__ void store16(uint16_t* p, const uint4& v) {
  const u32x4_t x = {v.x, v.y, v.z, v.w};
  if constexpr (NT) __builtin_nontemporal_store(x, reinterpret_cast<u32x4_t*>(p));
  else *reinterpret_cast<u32x4_t*>(p) = x;
}

// D a multiple of 16 with everything on 16 bytes: a group of LPG lanes (the power of two from D / 16 on)
// per token and HPT heads (q, then k, then with a cache v, which is only copied), lane l holding pairs
// 8l..8l+7, so that rotation needs no exchange, the norm one sum over the group, and the table entries
// (chosen by axis) are read once for all HPT heads.  LD, ST: heads read, written with the non-temporal hint.
template <int LPG, int HPT, bool LD, bool ST, class TAB>
__global__ __launch_bounds__(256) void qk_norm_mrope_vec_kernel(MropeArgs a, uint32_t groups) {
  EZ_PROF_WAVE(kProfQkMrope);
  const int l = threadIdx.x % LPG;
  const uint32_t g = blockIdx.x * (256 / LPG) + threadIdx.x / LPG;
  const uint32_t tok = g / groups;
  const int u0 = int(g - tok * groups) * HPT, half = a.D / 2;
  const int heads = a.H + a.Hkv, units = heads + (a.Kc ? a.Hkv : 0);
  const int64_t t = tok;
  if (t >= a.T) return;
  const bool lane_on = 8 * l < half;  // lanes behind the head's last pair only join the sums
  const int at = lane_on ? 8 * l : 0;
  uint4 x1[HPT], x2[HPT];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int u = min(u0 + i, units - 1);
    const uint16_t* src = at + (u < a.H     ? a.q + t * a.q_rs + int64_t(u) * a.D
                                : u < heads ? a.k + t * a.k_rs + int64_t(u - a.H) * a.D
                                            : a.v + t * a.v_rs + int64_t(u - heads) * a.D);
    x1[i] = load16<LD>(src);
    x2[i] = load16<LD>(src + half);
  }
  int pos[kMaxAxes];
  bool ok = true;
#pragma unroll
  for (int n = 0; n < kMaxAxes; ++n) {
    pos[n] = n < a.A ? a.positions[n * a.T + t] : 0;
    ok &= pos[n] >= 0 && pos[n] < a.S;
  }
  const int64_t slot = a.Kc ? a.slots[t] : -1;
  const bool cached = slot >= 0 && slot < a.num_slots;
  if (!ok) return;  // the whole group

  float c[8], s[8];
  load8(static_cast<const TAB*>(a.cos) + int64_t(pos[0]) * a.D + at, c);
  load8(static_cast<const TAB*>(a.sin) + int64_t(pos[0]) * a.D + at, s);
  if (a.A > 1) {
    int ax[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) ax[e] = axis_of(a, at + e);
#pragma unroll
    for (int n = 1; n < kMaxAxes; ++n) {
      if (n < a.A) {
        float cn[8], sn[8];
        load8(static_cast<const TAB*>(a.cos) + int64_t(pos[n]) * a.D + at, cn);
        load8(static_cast<const TAB*>(a.sin) + int64_t(pos[n]) * a.D + at, sn);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          c[e] = ax[e] == n ? cn[e] : c[e];
          s[e] = ax[e] == n ? sn[e] : s[e];
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int u = u0 + i;  // the group as a whole has it or not
    const bool is_q = u < a.H;
    uint4 p1 = x1[i], p2 = x2[i];
    if (u < heads) {
      float y1[8], y2[8];
      unpack8(x1[i], y1);
      unpack8(x2[i], y2);
      if (a.norm) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += y1[e] * y1[e] + y2[e] * y2[e];
        const float r = rsqrtf(group_sum<LPG>(lane_on ? ss : 0.f) / float(a.D) + a.eps);
        const uint16_t* w = is_q ? a.qw : a.kw;
        float w1[8], w2[8];
        if (w) {
          load8(w + at, w1);
          load8(w + at + half, w2);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y1[e] = __fmul_rn(y1[e], r);
          y2[e] = __fmul_rn(y2[e], r);
          if (w) {
            y1[e] = __fmul_rn(y1[e], w1[e]);
            y2[e] = __fmul_rn(y2[e], w2[e]);
          }
        }
      }
      float o1[8], o2[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        o1[e] = __fadd_rn(__fmul_rn(y1[e], c[e]), __fmul_rn(-y2[e], s[e]));
        o2[e] = __fadd_rn(__fmul_rn(y2[e], c[e]), __fmul_rn(y1[e], s[e]));
      }
      p1 = make_uint4(pack_bf2(o1[0], o1[1]), pack_bf2(o1[2], o1[3]), pack_bf2(o1[4], o1[5]), pack_bf2(o1[6], o1[7]));
      p2 = make_uint4(pack_bf2(o2[0], o2[1]), pack_bf2(o2[2], o2[3]), pack_bf2(o2[4], o2[5]), pack_bf2(o2[6], o2[7]));
    }
    if (lane_on && u < units) {
      uint16_t* dst = is_q ? a.q_out + (t * a.H + u) * a.D : a.k_out && u < heads ? a.k_out + (t * a.Hkv + u - a.H) * a.D : nullptr;
      if (dst) {
        store16<ST>(dst + at, p1);
        store16<ST>(dst + at + half, p2);
      }
      if (!is_q && cached) {
        uint16_t* pool = u < heads ? a.Kc + slot_offset(a, slot, u - a.H) : a.Vc + slot_offset(a, slot, u - heads);
        store16<ST>(pool + at, p1);
        store16<ST>(pool + at + half, p2);
      }
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool vec_form(const MropeArgs& a) {
  return a.D % 16 == 0 && a.q_rs % 8 == 0 && a.k_rs % 8 == 0 && a.v_rs % 8 == 0 && aligned16(a.q) && aligned16(a.k) &&
         aligned16(a.v) && aligned16(a.qw) && aligned16(a.kw) && aligned16(a.cos) && aligned16(a.sin) && aligned16(a.Kc) &&
         aligned16(a.Vc) && aligned16(a.q_out) && aligned16(a.k_out) && a.T * (a.H + 2 * a.Hkv) < (int64_t(1) << 31);
}

template <int LPG, int HPT, bool LD, bool ST>
void launch_vec(const MropeArgs& a, hipStream_t s) {
  const uint32_t groups = uint32_t((a.H + (a.Kc ? 2 : 1) * a.Hkv + HPT - 1) / HPT);
  const dim3 grid(unsigned((a.T * groups + 256 / LPG - 1) / (256 / LPG)));
  if (a.table_f32) hipLaunchKernelGGL((qk_norm_mrope_vec_kernel<LPG, HPT, LD, ST, float>), grid, dim3(256), 0, s, a, groups);
  else hipLaunchKernelGGL((qk_norm_mrope_vec_kernel<LPG, HPT, LD, ST, uint16_t>), grid, dim3(256), 0, s, a, groups);
}

// The non-temporal hint, by the bytes of the heads read and written.  From 8 MB on where half a head is whole lines
// of 128 bytes (1024 / 4097 / 16384 tokens of 16 + 2 x 8, 16 + 2 x 8 and 32 + 2 x 8 heads of 128: 9.1 / 21.6 / 92 us
// without, 7.3 / 16.4 / 80 with it; a copy that reads q_out afterwards included, 11.7 / 27.7 and 11.4 / 25.8; 256
// tokens with that copy 7.7 and 7.5, 128 tokens 6.9 and 7.4).  Where the halves of a head share lines, never on the
// loads, which would fetch them twice (20000 tokens of 16 + 16 heads of 80: 61 us without, 70 with it), and on the
// stores up to the size of the L2s, twice that where the heads are whole lines (3000 tokens 15.1 and 12.8 us, with the
// copy 19.0 and 17.9, but for 6000 tokens 30.7 and 33.4; 4097 tokens of 32 + 2 x 8 heads of 64 18.2 and 14.6, with it
// 24.8 and 23.6, for 8192 44.1 and 44.3).
template <int LPG, int HPT>
void launch_vec(const MropeArgs& a, int64_t heads, hipStream_t s) {
  const int64_t bytes = a.T * heads * a.D * 4;
  if (bytes >= int64_t(8) << 20) {
    if constexpr (LPG >= 8)  // heads of at least 128
      if (a.D % 128 == 0) return launch_vec<LPG, HPT, true, true>(a, s);
    if (a.D % 128 != 0 && bytes < int64_t(a.D % 64 == 0 ? 64 : 32) << 20) return launch_vec<LPG, HPT, false, true>(a, s);
  }
  launch_vec<LPG, HPT, false, false>(a, s);
}

template <int LPG>
void launch_vec(const MropeArgs& a, hipStream_t s) {
  const int64_t heads = a.H + (a.Kc ? 2 : 1) * a.Hkv;
  // Four heads a group once that still gives every CU 512 threads (16 + 2 x 8 heads of 128: 1400 tokens take 8.8 us
  // with one head a group and 10.0 with four, 3000 tokens 15.3 and 13.4).
  if (a.T * heads * LPG < int64_t(8) * 256 * 256) launch_vec<LPG, 1>(a, heads, s);
  else launch_vec<LPG, 4>(a, heads, s);
}

int launch_mrope(const MropeArgs& a, hipStream_t s) {
  if (vec_form(a)) {
    if (a.D <= 64) launch_vec<4>(a, s);
    else if (a.D <= 128) launch_vec<8>(a, s);
    else if (a.D <= 256) launch_vec<16>(a, s);
    else launch_vec<32>(a, s);
    return launch_status("qk_norm_mrope");
  }
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
  // q_out in q's place and k_out in k's are fine (every lane reads what it writes first), other overlaps a race
  auto span = [&](int64_t rs, int64_t heads) { return ((T - 1) * rs + heads * D) * 2; };
  const int64_t nq = T * H * D * 2, nk = T * Hkv * D * 2;
  EZ_REQUIRE((q_out == q && q_stride == H * D) || !ez::overlap(q_out, nq, q, span(q_stride, H)),
             "qk_norm_mrope: q_out must be q (tokens next to each other) or not overlap it");
  EZ_REQUIRE((k_out == k && k_stride == Hkv * D) || !ez::overlap(k_out, nk, k, span(k_stride, Hkv)),
             "qk_norm_mrope: k_out must be k (tokens next to each other) or not overlap it");
  EZ_REQUIRE(!ez::overlap(q_out, nq, k, span(k_stride, Hkv)) && !ez::overlap(q_out, nq, k_out, nk) &&
                 !ez::overlap(k_out, nk, q, span(q_stride, H)) &&
                 !(K_cache && (ez::overlap(q_out, nq, v, span(v_stride, Hkv)) || ez::overlap(k_out, nk, v, span(v_stride, Hkv)))),
             "qk_norm_mrope: an output overlaps another tensor");
  const int64_t pool = a.num_slots * Hkv * D * 2;  // 0 without a cache
  for (const void* c : {K_cache, V_cache})
    EZ_REQUIRE(!ez::overlap(c, pool, q, span(q_stride, H)) && !ez::overlap(c, pool, k, span(k_stride, Hkv)) &&
                   !ez::overlap(c, pool, v, span(v_stride, Hkv)) && !ez::overlap(c, pool, q_out, nq) &&
                   !ez::overlap(c, pool, k_out, nk),
               "qk_norm_mrope: a cache overlaps another tensor");
  EZ_REQUIRE(!ez::overlap(K_cache, pool, V_cache, pool), "qk_norm_mrope: K_cache and V_cache overlap");
  const int64_t table = S * D * (table_f32 ? 4 : 2);
  const struct { const void* p; int64_t n; } small[] = {{cos, table}, {sin, table}, {positions, axes * T * 4},
      {K_cache ? slot_mapping : nullptr, T * 8}, {norm ? q_norm_w : nullptr, D * 2}, {norm ? k_norm_w : nullptr, D * 2}};
  for (const auto& x : small)
    EZ_REQUIRE(!ez::overlap(x.p, x.n, q_out, nq) && !ez::overlap(x.p, x.n, k_out, nk) &&
                   !ez::overlap(x.p, x.n, K_cache, pool) && !ez::overlap(x.p, x.n, V_cache, pool),
               "qk_norm_mrope: an output overlaps a table, the positions, the slots or a weight");
  return ez::launch_mrope(a, stream);
}
