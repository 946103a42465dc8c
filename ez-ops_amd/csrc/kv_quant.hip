// Cache rows into 8 bits and back, by slot.
//
// Quantise: a run of consecutive slots inside one block of tokens (all the new
// tokens that the block gets in this call) is one unit per kv head and per K / V:
//   need = least e with max |x| <= TOP 2^e over the run
//   e    = need, where the run begins the block (its first row); else max(need, e_old),
//          and the rows before the run become round(code 2^(e_old - e)) if e > e_old
//   code = round(x 2^-e)
// so every row is rounded against the scale that its block has after the call.
//
// Both directions are memory traffic: 2 bytes a value in, 1 out, or the reverse.  A unit
// is one wave (blocks of few rows) or the four or eight waves of a block: the run's
// rows are read once, whole rows by 16-byte loads, and wait in registers (32 at most) for
// the maximum over all of them.  A wave looks at a window of tokens: one
// load of 64 slots tells which of them begin a run and how long it is; runs of one token
// (a decode step) go several to a wave, a row to each 8 or 16 lanes.
//
// Measured: 16384 tokens of 8 heads of 128 written in 18 us and read back in 16
// where the memory-side cache holds some of them; 45 us a call of both on inputs that no
// cache holds (a large copy of as many bytes 39).  40000 rows read back in 51 us, 5.0 TB/s
// (copy 5.1).  64 single tokens 3.3 us, a launch and two dependent loads, where no scale grows;
// where one does, the 8 or 16 lanes of the row turn the block's earlier rows 4 bytes each at a
// time: all 64 at the last row of their block 17 us in blocks of 32 rows, 130 to 140 in blocks of
// 256, 155 to 195 with heads of 64.
#include "common.h"
#include "internal.h"
#include "kv8.h"
#include "prof.h"
#include "status.h"
#include "../../include/ezops_hip.h"

namespace ez {

EZ_PROF_DEFINE(kvquant)
namespace {

struct KvQuantArgs {
  Kv8Args c;
  const uint16_t *k, *v;   // [T, Hkv, D], tokens k_rs / v_rs elements apart
  int64_t k_rs, v_rs;
  const int64_t* slots;    // [T]
  int64_t T;
};

struct KvDequantArgs {
  Kv8Args c;
  const int64_t* slots;    // [T]
  uint16_t *k_out, *v_out;  // [T, Hkv, D]
  int64_t T;
};

__device__ __forceinline__ bool slot_ok(int64_t s, int64_t n) { return s >= 0 && s < n; }

__device__ __forceinline__ uint32_t pk_max_u16(uint32_t a, uint32_t b) {
  typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t,
                            __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#define EZ_DPP_STEP(ctrl) v = max(v, uint32_t(__builtin_amdgcn_mov_dpp(int(v), ctrl, 0xF, 0xF, true)));
  EZ_DPP_STEP(0xB1)   // quad_perm [1,0,3,2]
  EZ_DPP_STEP(0x4E)   // quad_perm [2,3,0,1]
  EZ_DPP_STEP(0x141)  // row_half_mirror
  EZ_DPP_STEP(0x140)  // row_mirror
#undef EZ_DPP_STEP
  const uint32_t a = max(uint32_t(__builtin_amdgcn_readlane(int(v), 0)), uint32_t(__builtin_amdgcn_readlane(int(v), 16)));
  const uint32_t b = max(uint32_t(__builtin_amdgcn_readlane(int(v), 32)), uint32_t(__builtin_amdgcn_readlane(int(v), 48)));
  return max(a, b);
}

// 8 values -> codes of scale 2^(e - 127).  Values that are finite and inside the scale (but
// for one at the upper end of scales) take the short conversion.
template <int TYPE>
__device__ __forceinline__ uint2 to_codes(const uint4& x, int e, bool finite) {
  if (finite && e < kKvHighExp) return kv8_codes8<TYPE>(x, e);
  const float inv = e == kKvNanExp ? 0.f : __uint_as_float(uint32_t(254 - e) << 23);
  float f[8];
  unpack8(x, f);
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = TYPE == kKvInt8 && e == kKvNanExp ? 0.f : f[k] * inv;
  const float lo[4] = {f[0], f[1], f[2], f[3]}, hi[4] = {f[4], f[5], f[6], f[7]};
  return make_uint2(kv8_codes<TYPE>(lo), kv8_codes<TYPE>(hi));
}

// The n rows a block held before, from scale `old` to the larger e: 4 codes a lane, `of` lanes.
template <int D, int TYPE>
__device__ __forceinline__ void turn_rows(uint8_t* rows, int n, int old, int e, int lane, int of) {
  const float r = e == kKvNanExp ? 0.f : __uint_as_float(uint32_t(127 + old - e) << 23);
  uint32_t* held = reinterpret_cast<uint32_t*>(rows);
  for (int i = lane; i < n * D / 4; i += of) {
    float y[4];
    kv8_f32x4<TYPE>(held[i], y);
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] *= r;
    held[i] = kv8_codes<TYPE>(y);
  }
}

// Rows [t, t + n) of one head into the block that holds slot `slot`, WPU waves together,
// `part` of them this one; CH rows a wave (n <= CH WPU).
template <int D, int TYPE, int CH, int WPU>
__device__ __forceinline__ void quant_run(const KvQuantArgs& a, int64_t t, int64_t slot, int n, int h, bool is_v, int part,
                                          uint32_t* shared_max) {
  constexpr int LPR = D / 8, RPI = kWave / LPR, NI = CH / RPI;  // lanes of a row, rows of a load, loads
  const int lane = threadIdx.x & (kWave - 1);
  const int off = int(slot) & ((1 << a.c.block_sh) - 1);
  const int64_t rs = is_v ? a.v_rs : a.k_rs;
  const uint16_t* src = (is_v ? a.v : a.k) + t * rs + int64_t(h) * D + lane % LPR * 8;
  const int64_t row0 = (((slot >> a.c.page_sh) * a.c.Hkv + h) << a.c.page_sh) + (slot & ((int64_t(1) << a.c.page_sh) - 1));
  uint8_t* sp = (is_v ? a.c.Vs : a.c.Ks) + (row0 >> a.c.block_sh);
  uint8_t* dst = (is_v ? a.c.V : a.c.K) + row0 * D;
  const int r0 = part * CH + lane / LPR;
  int old = off ? int(*sp) : 0;
  uint4 x[NI];
  uint32_t m2 = 0;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    x[i] = make_uint4(0, 0, 0, 0);
    if (part * CH + i * RPI < n) {
      const int r = r0 + i * RPI;
      if (r < n) x[i] = *reinterpret_cast<const uint4*>(src + r * rs);
    }
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const uint32_t mask = 0x7fff7fffu;
    const uint4 v = x[i];
    m2 = pk_max_u16(m2, pk_max_u16(pk_max_u16(v.x & mask, v.y & mask), pk_max_u16(v.z & mask, v.w & mask)));
  }
  auto all_waves = [&](uint32_t m) {
    m = wave_max_u32(m);
    if constexpr (WPU > 1) {
      if (lane == 0) shared_max[part] = m;
      __syncthreads();
      for (int w = 0; w < WPU; ++w) m = max(m, shared_max[w]);
      __syncthreads();
    }
    return uint32_t(__builtin_amdgcn_readfirstlane(int(m)));
  };
  old = kv8_exp(__builtin_amdgcn_readfirstlane(old));  // here, before a wave that is done may write the new one
  uint32_t m = all_waves(max(m2 & 0xffffu, m2 >> 16));
  const bool finite = m < 0x7f80u;
  if (TYPE == kKvE4m3 && !finite) {  // the finite values alone set the scale
    m = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t lo = w[k] & 0x7fffu, hi = (w[k] >> 16) & 0x7fffu;
        m = max(m, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
      }
    }
    m = all_waves(m);
  }
  int e = TYPE == kKvInt8 && !finite ? kKvNanExp : kv8_need<TYPE>(m);
  if (off) {
    e = max(e, old);
    if (e > old) turn_rows<D, TYPE>(dst - int64_t(off) * D, off, old, e, part * kWave + lane, WPU * kWave);
  }
#pragma unroll
  for (int i = 0; i < NI; ++i)
    if (part * CH + i * RPI < n) {
      const int r = r0 + i * RPI;
      const uint2 w = to_codes<TYPE>(x[i], e, finite);
      if (r < n) *reinterpret_cast<uint2*>(dst + r * D + lane % LPR * 8) = w;
    }
  if (lane == 0 && part == 0) *sp = uint8_t(e);
}

// Runs of one token: the lanes of a row (D / 8) take one each, so a wave takes RPI of them
// at a time.  Token `t` goes to `slot`, where these lanes have one (`on`).
template <int D, int TYPE>
__device__ __forceinline__ void quant_singles(const KvQuantArgs& a, int64_t t, int64_t slot, bool on, int h, bool is_v) {
  constexpr int LPR = D / 8;
  const int c = threadIdx.x % LPR;
  uint8_t *sp = nullptr, *dst = nullptr;
  uint4 x = make_uint4(0, 0, 0, 0);
  int off = 0, old = 0;
  if (on) {
    off = int(slot) & ((1 << a.c.block_sh) - 1);
    const int64_t row0 = (((slot >> a.c.page_sh) * a.c.Hkv + h) << a.c.page_sh) + (slot & ((int64_t(1) << a.c.page_sh) - 1));
    sp = (is_v ? a.c.Vs : a.c.Ks) + (row0 >> a.c.block_sh);
    dst = (is_v ? a.c.V : a.c.K) + row0 * D;
    x = *reinterpret_cast<const uint4*>((is_v ? a.v + t * a.v_rs : a.k + t * a.k_rs) + int64_t(h) * D + 8 * c);
    old = off ? kv8_exp(int(*sp)) : 0;
  }
  auto row_max = [](uint32_t v) {
#define EZ_DPP_STEP(ctrl) v = max(v, uint32_t(__builtin_amdgcn_mov_dpp(int(v), ctrl, 0xF, 0xF, true)));
    EZ_DPP_STEP(0xB1)
    EZ_DPP_STEP(0x4E)
    EZ_DPP_STEP(0x141)
    if constexpr (LPR == 16) { EZ_DPP_STEP(0x140) }
#undef EZ_DPP_STEP
    return v;
  };
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) m = max(m, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
  m = row_max(m);
  const bool finite = m < 0x7f80u;
  if (TYPE == kKvE4m3 && __ballot(!finite)) {  // the finite values alone set the scale
    uint32_t f = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t lo = w[k] & 0x7fffu, hi = (w[k] >> 16) & 0x7fffu;
      f = max(f, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
    }
    m = row_max(f);
  }
  if (!on) return;
  const int e = max(TYPE == kKvInt8 && !finite ? kKvNanExp : kv8_need<TYPE>(m), old);
  if (off && e > old) turn_rows<D, TYPE>(dst - int64_t(off) * D, off, old, e, c, LPR);
  *reinterpret_cast<uint2*>(dst + 8 * c) = to_codes<TYPE>(x, e, finite);
  if (c == 0) *sp = uint8_t(e);
}

template <int D, int TYPE, int CH, int WPU>
__global__ __launch_bounds__(WPU > 4 ? WPU * kWave : 256) void kv_quant_kernel(KvQuantArgs a, int window) {
  EZ_PROF_WAVE(kProfKvQuant);
  constexpr int LPR = D / 8, RPI = kWave / LPR;
  __shared__ uint32_t shared_max[WPU];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t u = WPU == 1 ? int64_t(blockIdx.x) * 4 + wave : int64_t(blockIdx.x);
  const int units = 2 * a.c.Hkv;  // of a window
  const int64_t t0 = u / units * window;
  if (t0 >= a.T) return;
  const int hv = int(u % units), h = hv >> 1;
  // Lane i holds the slot of token t0 + i.
  const int64_t ti = t0 + lane;
  const int64_t s = ti < a.T ? a.slots[ti] : -1;
  const int64_t back = t0 > 0 ? a.slots[t0 - 1] : -1;
  const bool ok = slot_ok(s, a.c.num_slots);
  const int64_t up = __shfl_up(s, 1, kWave), before = lane ? up : back;
  const int bmask = (1 << a.c.block_sh) - 1;
  // tokens that go on with the run of the token before them
  const uint64_t cont = __ballot(ok && slot_ok(before, a.c.num_slots) && before + 1 == s && (int(s) & bmask) != 0);
  const uint64_t mine = window == 64 ? ~uint64_t(0) : (uint64_t(1) << window) - 1;
  const uint64_t first = __ballot(ok) & ~cont & mine;
  // a run of one token, but for one that ends where the slots at hand end
  uint64_t single = first & ~(cont >> 1) & ~(uint64_t(1) << 63);
  uint64_t many = first & ~single;
  for (int p = 0; single; ++p) {
    int i = -1;
#pragma unroll
    for (int g = 0; g < RPI; ++g) {
      if (single && lane / LPR == g) i = __ffsll(static_cast<unsigned long long>(single)) - 1;
      single &= single - 1;
    }
    const int64_t slot = __shfl(s, i < 0 ? 0 : i, kWave);
    if (p % WPU == (WPU == 1 ? 0 : wave)) quant_singles<D, TYPE>(a, t0 + i, slot, i >= 0, h, hv & 1);
  }
  while (many) {
    const int i = __ffsll(static_cast<unsigned long long>(many)) - 1;
    many &= many - 1;
    const int64_t t = t0 + i;
    const uint64_t sb = uint64_t(s);
    const int64_t slot = int64_t(uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(sb)), i))) |
                                 uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(sb >> 32)), i))) << 32);
    const uint64_t after = i < 63 ? ~(cont >> (i + 1)) : ~uint64_t(0);
    int n = min(__ffsll(static_cast<unsigned long long>(after)), 64 - i);
    if (i + n == 64) {  // the run may go on behind the slots at hand
      const int most = int(min(int64_t(bmask + 1 - (int(slot) & bmask)), a.T - t));
      while (n < most) {
        const int r = n + lane;
        const uint64_t same = __ballot(r < most && a.slots[t + min(r, most - 1)] == slot + r);
        const int more = ~same ? __ffsll(static_cast<unsigned long long>(~same)) - 1 : 64;
        n += more;
        if (more < 64) break;
      }
    }
    quant_run<D, TYPE, CH, WPU>(a, t, slot, n, h, hv & 1, WPU == 1 ? 0 : wave, shared_max);
  }
}

// Rows back to bf16: 8 values a thread and tensor, kPer of them in flight.
template <int D, int TYPE>
__global__ __launch_bounds__(256) void kv_dequant_kernel(KvDequantArgs a, int tokens) {
  EZ_PROF_WAVE(kProfKvDequant);
  constexpr int kPer = 4;
  const int cpt = a.c.Hkv * (D / 8);  // 16-byte pieces of a token's row
  const int64_t t0 = int64_t(blockIdx.x) * tokens;
  const int total = int(min(int64_t(tokens), a.T - t0)) * cpt;
  for (int i0 = threadIdx.x; i0 < total; i0 += kPer * 256) {
    uint2 k[kPer], v[kPer];
    int ek[kPer], ev[kPer];
    bool on[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = min(i0 + j * 256, total - 1);
      const int t = i / cpt, c = i - t * cpt, h = c / (D / 8), d = c % (D / 8) * 8;
      const int64_t slot = a.slots[t0 + t];
      on[j] = slot_ok(slot, a.c.num_slots) && i0 + j * 256 < total;
      const int64_t s = on[j] ? slot : 0;
      const int64_t at = (((s >> a.c.page_sh) * a.c.Hkv + h) << a.c.page_sh) + (s & ((int64_t(1) << a.c.page_sh) - 1));
      k[j] = *reinterpret_cast<const uint2*>(a.c.K + at * D + d);
      v[j] = *reinterpret_cast<const uint2*>(a.c.V + at * D + d);
      ek[j] = a.c.Ks[at >> a.c.block_sh];
      ev[j] = a.c.Vs[at >> a.c.block_sh];
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      auto wide = [](const uint2& w, int e) {
        const float s = kv8_scale(e);
        float y[4], z[4];
        kv8_f32x4<TYPE>(w.x, y);
        kv8_f32x4<TYPE>(w.y, z);
        return make_uint4(cvt_bf2(y[0] * s, y[1] * s), cvt_bf2(y[2] * s, y[3] * s), cvt_bf2(z[0] * s, z[1] * s),
                          cvt_bf2(z[2] * s, z[3] * s));
      };
      if (on[j]) {
        const int64_t out = t0 * cpt + i0 + j * 256;
        reinterpret_cast<uint4*>(a.k_out)[out] = wide(k[j], ek[j]);
        reinterpret_cast<uint4*>(a.v_out)[out] = wide(v[j], ev[j]);
      }
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_rows(const char* op, int64_t T, int64_t Hkv, int64_t D) {
  EZ_REQUIRE(T >= 1 && T < (int64_t(1) << 30), "%s: tokens must be in [1, 2^30)", op);
  EZ_REQUIRE(Hkv >= 1 && Hkv <= 4096, "%s: num_kv_heads must be in [1, 4096]", op);
  EZ_REQUIRE(D == 64 || D == 128, "%s: head_dim must be 64 or 128", op);
  return EZ_OK;
}

}  // namespace
}  // namespace ez

extern "C" int ezops_kv_cache_quant_bf16(const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                                         const int64_t* slot_mapping, void* K_cache, void* V_cache, void* K_scale,
                                         void* V_scale, int cache_type, int64_t num_pages, int64_t page_size,
                                         int64_t block_size, int64_t T, int64_t Hkv, int64_t D, hipStream_t stream) {
  const char* op = "kv_cache_quant";
  EZ_REQUIRE(k && v && slot_mapping, "%s: null pointer", op);
  int rc = ez::check_rows(op, T, Hkv, D);
  if (rc != EZ_OK) return rc;
  ez::KvQuantArgs a{};
  ez::fill_kv8(a.c, K_cache, V_cache, K_scale, V_scale, cache_type, num_pages, page_size, block_size, Hkv, D);
  rc = ez::check_kv8(op, a.c, page_size, block_size);
  if (rc != EZ_OK) return rc;
  EZ_REQUIRE(k_stride >= Hkv * D && v_stride >= Hkv * D, "%s: token strides below the heads' size", op);
  EZ_REQUIRE(k_stride % 8 == 0 && v_stride % 8 == 0 && ez::aligned16(k) && ez::aligned16(v),
             "%s: rows of k and v must begin at multiples of 16 bytes", op);
  const int64_t pool = ez::kv8_pool_bytes(a.c), sc = ez::kv8_scale_bytes(a.c);
  const struct { const void* p; int64_t n; } out[] = {{K_cache, pool}, {V_cache, pool}, {K_scale, sc}, {V_scale, sc}},
      in[] = {{k, ((T - 1) * k_stride + Hkv * D) * 2}, {v, ((T - 1) * v_stride + Hkv * D) * 2}, {slot_mapping, T * 8}};
  for (int i = 0; i < 4; ++i) {
    for (const auto& x : in) EZ_REQUIRE(!ez::overlap(out[i].p, out[i].n, x.p, x.n), "%s: a cache overlaps an input", op);
    for (int j = 0; j < i; ++j)
      EZ_REQUIRE(!ez::overlap(out[i].p, out[i].n, out[j].p, out[j].n), "%s: caches and scales overlap", op);
  }
  a.k = static_cast<const uint16_t*>(k); a.k_rs = k_stride;
  a.v = static_cast<const uint16_t*>(v); a.v_rs = v_stride;
  a.slots = slot_mapping; a.T = T;
  // Tokens that the waves of a unit look at: doubled up to 64 while there are more than 4096
  // units (a window, a kv head, K or V), so that 2049 to 4096 are left.  In a prompt most
  // tokens begin no run, and a wave that finds none still holds its place for two loads; few
  // tokens want many waves.  The kernel alone, 8 heads of 128, at 8, 16, 32 and 64 tokens:
  // 16384 tokens in blocks of 32 rows 34, 26, 18 and 17 us, of 64 33, 24, 20 and 17.5, of 256 65,
  // 44, 33 and 27 (the rule: 64); a mixed step of 3684 tokens in blocks of 16 7.5, 6.9, 7.8 and
  // 10.2, of 64 10.8, 8.6, 8.0 and 8.4 (16).  Between these it is not the best: 4096 tokens of one
  // prompt 8.8 us at its 16, 5.9 at 32; 1024 5.8 at its 4, 4.4 at 16.
  int window = 1;
  while (window < 64 && T * Hkv * 2 / window > 4096) window *= 2;
  const int64_t units = (T + window - 1) / window * Hkv * 2;
  // Rows of a wave and waves of a run: 32 registers of values a lane at most, and 16 where
  // four waves hold a whole block in that (16384 tokens of heads of 128 in blocks of 64: two
  // waves a SIMD with 64 registers 50.6 us with the read-back, 45 so; three prompts of 5250
  // in blocks of 256 53.4, with eight waves 51).  Rows of heads of 64 have half the bytes: the
  // same two cases 28.4 and 35.5 us with as many waves, 26.6 and 31.3 with one and four, 64
  // rows each.
#define EZ_RUN(DD, TY, CH, WPU)                                                                              \
  do {                                                                                                       \
    constexpr int threads = (WPU) > 4 ? (WPU) * 64 : 256;                                                    \
    const int64_t blocks = (WPU) == 1 ? (units + 3) / 4 : units;                                             \
    EZ_REQUIRE(blocks < (int64_t(1) << 32) / threads, "%s: tokens * heads past one launch", op);             \
    hipLaunchKernelGGL((ez::kv_quant_kernel<DD, TY, CH, WPU>), dim3(unsigned(blocks)), dim3(threads), 0, stream, a, window); \
  } while (0)
#define EZ_GO(DD, TY)                                                                      \
  do {                                                                                     \
    if (block_size <= 32) EZ_RUN(DD, TY, 32, 1);                                           \
    else if (block_size == 64) EZ_RUN(DD, TY, (DD == 64 ? 64 : 16), (DD == 64 ? 1 : 4));   \
    else if (block_size == 128) EZ_RUN(DD, TY, 32, 4);                                     \
    else EZ_RUN(DD, TY, (DD == 64 ? 64 : 32), (DD == 64 ? 4 : 8));                         \
  } while (0)
  EZ_KV8_DISPATCH(EZ_GO);
#undef EZ_GO
#undef EZ_RUN
  return ez::launch_status(op);
}

extern "C" int ezops_kv_cache_dequant_bf16(const void* K_cache, const void* V_cache, const void* K_scale,
                                           const void* V_scale, const int64_t* slot_mapping, int cache_type,
                                           int64_t num_pages, int64_t page_size, int64_t block_size, void* k_out,
                                           void* v_out, int64_t T, int64_t Hkv, int64_t D, hipStream_t stream) {
  const char* op = "kv_cache_dequant";
  EZ_REQUIRE(slot_mapping && k_out && v_out, "%s: null pointer", op);
  int rc = ez::check_rows(op, T, Hkv, D);
  if (rc != EZ_OK) return rc;
  ez::KvDequantArgs a{};
  ez::fill_kv8(a.c, K_cache, V_cache, K_scale, V_scale, cache_type, num_pages, page_size, block_size, Hkv, D);
  rc = ez::check_kv8(op, a.c, page_size, block_size);
  if (rc != EZ_OK) return rc;
  EZ_REQUIRE(ez::aligned16(k_out) && ez::aligned16(v_out), "%s: outputs must be 16-byte aligned", op);
  const int64_t pool = ez::kv8_pool_bytes(a.c), sc = ez::kv8_scale_bytes(a.c), nb = T * Hkv * D * 2;
  const struct { const void* p; int64_t n; } in[] = {{K_cache, pool}, {V_cache, pool}, {K_scale, sc}, {V_scale, sc},
                                                     {slot_mapping, T * 8}};
  for (const auto& x : in)
    EZ_REQUIRE(!ez::overlap(x.p, x.n, k_out, nb) && !ez::overlap(x.p, x.n, v_out, nb), "%s: an output overlaps an input", op);
  EZ_REQUIRE(!ez::overlap(k_out, nb, v_out, nb), "%s: the outputs overlap", op);
  a.slots = slot_mapping; a.T = T;
  a.k_out = static_cast<uint16_t*>(k_out); a.v_out = static_cast<uint16_t*>(v_out);
  const int cpt = int(Hkv * (D / 8));
  const int tokens = cpt >= 1024 ? 1 : 1024 / cpt;  // of a block: 4 pieces a thread
  const int64_t blocks = (T + tokens - 1) / tokens;
  EZ_REQUIRE(blocks < int64_t(1) << 24, "%s: tokens past one launch", op);
#define EZ_GO(DD, TY) hipLaunchKernelGGL((ez::kv_dequant_kernel<DD, TY>), dim3(unsigned(blocks)), dim3(256), 0, stream, a, tokens)
  EZ_KV8_DISPATCH(EZ_GO);
#undef EZ_GO
  return ez::launch_status(op);
}
