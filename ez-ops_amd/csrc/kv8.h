// The KV cache held in 8 bits, shared by its kernels.
//
// Pools: codes [num_pages, Hkv, page_size, D], int8 or OCP e4m3, and scales
// [num_pages, Hkv, page_size / block] of one byte each: the block's rows stand for
// code * 2^(e - 127) (E8M0; 255 = not a number).  Powers of two, because then
// x * 2^-e and code * 2^e are exact: a value is rounded once, the read-back is exact
// in bf16, and rows that are re-scaled when their block grows lose only the bits
// that leave the code.  An int8 row that was rounded at every growth of its block is
// off by less than 1/2 + 1/4 + ... < 1 step of the present scale; with scales of
// any size each small growth would add another half step.
#pragma once

#include "common.h"
#include "internal.h"
#include "status.h"

namespace ez {

enum KvType : int { kKvInt8 = 0, kKvE4m3 = 1 };

// Scales lie in 2^-60 .. 2^60: softmax weights times a scale, and divided by one,
// stay inside fp32 and bf16.  Larger values saturate, smaller ones become zero.
constexpr int kKvLowExp = 127 - 60, kKvHighExp = 127 + 60, kKvNanExp = 255;

struct Kv8Args {
  uint8_t *K, *V;        // codes
  uint8_t *Ks, *Vs;      // exponents
  int64_t num_pages, num_slots;
  int Hkv, D, type;
  int page_sh, block_sh;  // log2 of page_size and block
};

inline int check_kv8(const char* op, const Kv8Args& a, int64_t page_size, int64_t block) {
  EZ_REQUIRE(a.K && a.V && a.Ks && a.Vs, "%s: null pointer", op);
  EZ_REQUIRE(a.type == kKvInt8 || a.type == kKvE4m3, "%s: cache type must be int8 (0) or e4m3 (1)", op);
  EZ_REQUIRE(page_size >= 32 && page_size <= (1 << 20) && (page_size & (page_size - 1)) == 0 && a.num_pages >= 1 &&
                 a.num_pages < (int64_t(1) << 31) && a.num_slots <= (int64_t(1) << 40),
             "%s: page_size must be a power of two in [32, 2^20] and num_pages in [1, 2^31), 2^40 rows at most", op);
  EZ_REQUIRE(block >= 16 && block <= 256 && block <= page_size && (block & (block - 1)) == 0,
             "%s: block_size must be a power of two in [16, 256], at most page_size", op);
  EZ_REQUIRE(((reinterpret_cast<uintptr_t>(a.K) | reinterpret_cast<uintptr_t>(a.V)) & 15) == 0,
             "%s: caches must be 16-byte aligned", op);
  return EZ_OK;
}
inline void fill_kv8(Kv8Args& a, const void* K, const void* V, const void* Ks, const void* Vs, int type, int64_t num_pages,
                     int64_t page_size, int64_t block, int64_t Hkv, int64_t D) {
  auto mut = [](const void* p) { return static_cast<uint8_t*>(const_cast<void*>(p)); };
  a.K = mut(K); a.V = mut(V); a.Ks = mut(Ks); a.Vs = mut(Vs);
  a.type = type; a.num_pages = num_pages; a.Hkv = int(Hkv); a.D = int(D);
  a.page_sh = page_size > 0 ? __builtin_ctzll(static_cast<unsigned long long>(page_size)) : 0;
  a.block_sh = block > 0 ? __builtin_ctzll(static_cast<unsigned long long>(block)) : 0;
  a.num_slots = num_pages * page_size;
}
inline int64_t kv8_pool_bytes(const Kv8Args& a) { return a.num_slots * a.Hkv * a.D; }
inline int64_t kv8_scale_bytes(const Kv8Args& a) { return (a.num_slots >> a.block_sh) * a.Hkv; }

// Exponents outside [67, 187], which no write makes, are read as the nearest end; 255 stays.
__host__ __device__ __forceinline__ int kv8_exp(int e) {
  return e == kKvNanExp ? e : e < kKvLowExp ? kKvLowExp : e > kKvHighExp ? kKvHighExp : e;
}
// 2^(e - 127), NaN for 255.
__device__ __forceinline__ float kv8_scale(int e) {
  return __uint_as_float(e == kKvNanExp ? 0x7fc00000u : uint32_t(kv8_exp(e)) << 23);
}

// ---- codes -> bf16 (exact: e4m3 has 4 significant bits, int8 at most 7 and a sign)
template <int TYPE>
__device__ __forceinline__ uint2 kv8_bf16x4(uint32_t w) {
  if constexpr (TYPE == kKvE4m3) {
    return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(int(w), 1.f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(int(w), 1.f, true)));
  } else {  // one sign-extending byte conversion each
    const int x = int(w);
    return make_uint2(cvt_bf2(float(int8_t(x)), float(int8_t(x >> 8))), cvt_bf2(float(int8_t(x >> 16)), float(x >> 24)));
  }
}
template <int TYPE>
__device__ __forceinline__ void kv8_f32x4(uint32_t w, float (&f)[4]) {
  const uint2 p = kv8_bf16x4<TYPE>(w);
  f[0] = bf_lo(p.x); f[1] = bf_hi(p.x); f[2] = bf_lo(p.y); f[3] = bf_hi(p.y);
}

// ---- fp32 values in units of their scale -> codes, round to nearest even, saturating.
// Not finite: 0x7f in e4m3 (it has no infinities; the conversion itself makes 0xff of a
// NaN); int8 has no such code (its block's exponent says so).
template <int TYPE>
__device__ __forceinline__ uint32_t kv8_codes(const float (&y)[4]) {
  if constexpr (TYPE == kKvE4m3) {
    float c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = fminf(fmaxf(y[i], -448.f), 448.f);
    uint32_t w = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false));
    w = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], int(w), true));
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!(fabsf(y[i]) < INFINITY)) w = (w & ~(0xffu << (8 * i))) | (0x7fu << (8 * i));
    return w;
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int q = int(rintf(fminf(fmaxf(y[i], -127.f), 127.f)));
      w |= uint32_t(q & 255) << (8 * i);
    }
    return w;
  }
}

// Eight finite bf16 values of magnitude at most TOP 2^(e - 127) -> codes in scale 2^(e - 127).
// e4m3: one conversion with the scale for two values.  int8: x 2^-e + 1.5 2^23 leaves the
// nearest whole number, ties to even, in the low bits of the sum, as a signed byte.
template <int TYPE>
__device__ __forceinline__ uint2 kv8_codes8(const uint4& x, int e) {
  if constexpr (TYPE == kKvE4m3) {
    typedef short s16x2_t __attribute__((ext_vector_type(2)));
    const float s = __uint_as_float(uint32_t(e) << 23);
    s16x2_t lo{0, 0}, hi{0, 0};
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(lo, __builtin_bit_cast(bf16x2_t, x.x), s, false);
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(lo, __builtin_bit_cast(bf16x2_t, x.y), s, true);
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(hi, __builtin_bit_cast(bf16x2_t, x.z), s, false);
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(hi, __builtin_bit_cast(bf16x2_t, x.w), s, true);
    return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
  } else {
    const float inv = __uint_as_float(uint32_t(254 - e) << 23);
    float f[8];
    unpack8(x, f);
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(fmaf(f[i], inv, 12582912.f));
    auto pack = [](uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {
      const uint32_t lo = __builtin_amdgcn_perm(b1, b0, 0x0c0c0400u), hi = __builtin_amdgcn_perm(b3, b2, 0x0c0c0400u);
      return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
    };
    return make_uint2(pack(b[0], b[1], b[2], b[3]), pack(b[4], b[5], b[6], b[7]));
  }
}

// Least e with amax <= TOP 2^(e - 127) for the bf16 magnitude `m` (sign bit clear,
// finite): TOP = 127 = (1 + 126/128) 2^6 for int8, 448 = (1 + 96/128) 2^8 for e4m3.
template <int TYPE>
__device__ __forceinline__ int kv8_need(uint32_t m) {
  const int e = int(m >> 7), f = int(m & 127);
  const int n = TYPE == kKvInt8 ? e - 6 + (f > 126) : e - 8 + (f > 96);
  return min(max(n, kKvLowExp), kKvHighExp);
}

}  // namespace ez

// A launch for the head size D and the cache type of `a.c`.
#define EZ_KV8_DISPATCH(LAUNCH)                                      \
  do {                                                               \
    if (a.c.type == ez::kKvInt8) {                                   \
      if (D == 64) LAUNCH(64, ez::kKvInt8);                          \
      else LAUNCH(128, ez::kKvInt8);                                 \
    } else {                                                         \
      if (D == 64) LAUNCH(64, ez::kKvE4m3);                          \
      else LAUNCH(128, ez::kKvE4m3);                                 \
    }                                                                \
  } while (0)
