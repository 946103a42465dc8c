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
// One wave a unit: the wave that stands on a run's first token takes it, waves on
// other tokens leave after reading two slots.
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

template <int D, int TYPE>
__global__ __launch_bounds__(256) void kv_quant_kernel(KvQuantArgs a) {
  EZ_PROF_WAVE(kProfKvQuant);
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t units = a.T * a.c.Hkv * 2;
  for (int64_t u = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); u < units; u += int64_t(gridDim.x) * 4) {
    const bool is_v = u & 1;
    const int h = int((u >> 1) % a.c.Hkv);
    const int64_t t = (u >> 1) / a.c.Hkv;
    const int block = 1 << a.c.block_sh;
    const int64_t slot = a.slots[t];
    if (!slot_ok(slot, a.c.num_slots)) continue;
    const int off = int(slot & (block - 1));
    if (off != 0 && t > 0 && a.slots[t - 1] == slot - 1) continue;  // inside a run
    int n = 1;
    while (n < block - off && t + n < a.T && a.slots[t + n] == slot + n) ++n;

    const uint16_t* src = (is_v ? a.v + t * a.v_rs : a.k + t * a.k_rs) + int64_t(h) * D;
    const int64_t rs = is_v ? a.v_rs : a.k_rs;
    uint32_t m = 0;
    bool nan = false;
    for (int i = lane; i < n * D; i += kWave) {
      const uint32_t b = src[(i / D) * rs + i % D] & 0x7fffu;
      if (b >= 0x7f80u) nan = true;
      else m = max(m, b);
    }
    for (int o = 32; o > 0; o >>= 1) m = max(m, uint32_t(__shfl_xor(int(m), o, kWave)));
    const bool poison = TYPE == kKvInt8 && __ballot(nan) != 0;
    const int64_t page = slot >> a.c.page_sh;
    const int64_t row0 = ((page * a.c.Hkv + h) << a.c.page_sh) + (slot & ((int64_t(1) << a.c.page_sh) - 1));
    uint8_t* sp = (is_v ? a.c.Vs : a.c.Ks) + (row0 >> a.c.block_sh);
    uint8_t* dst = (is_v ? a.c.V : a.c.K) + row0 * D;
    const int old = off ? kv8_exp(int(*sp)) : 0;
    int e = poison ? kKvNanExp : kv8_need<TYPE>(m);
    e = max(e, old);
    if (off && e > old) {
      const float r = e == kKvNanExp ? 0.f : __uint_as_float(uint32_t(127 + old - e) << 23);
      uint32_t* old_rows = reinterpret_cast<uint32_t*>(dst - int64_t(off) * D);
      for (int i = lane; i < off * D / 4; i += kWave) {
        float y[4];
        kv8_f32x4<TYPE>(old_rows[i], y);
        for (int j = 0; j < 4; ++j) y[j] *= r;
        old_rows[i] = kv8_codes<TYPE, true>(y);
      }
    }
    const float inv = e == kKvNanExp ? 0.f : __uint_as_float(uint32_t(254 - e) << 23);
    for (int i = lane; i < n * D / 4; i += kWave) {
      const uint16_t* p = src + (4 * i / D) * rs + 4 * i % D;
      float y[4];
      for (int j = 0; j < 4; ++j) {
        y[j] = bf2f(p[j]) * inv;
        if (poison) y[j] = 0.f;
      }
      reinterpret_cast<uint32_t*>(dst)[i] = kv8_codes<TYPE, true>(y);
    }
    if (lane == 0) *sp = uint8_t(e);
  }
}

template <int D, int TYPE>
__global__ __launch_bounds__(256) void kv_dequant_kernel(KvDequantArgs a) {
  EZ_PROF_WAVE(kProfKvDequant);
  const int64_t n = a.T * a.c.Hkv * (D / 4);
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) {
    const int64_t row = i / (D / 4), t = row / a.c.Hkv;
    const int d = int(i % (D / 4)) * 4, h = int(row % a.c.Hkv);
    const int64_t slot = a.slots[t];
    if (!slot_ok(slot, a.c.num_slots)) continue;
    const int64_t at = (((slot >> a.c.page_sh) * a.c.Hkv + h) << a.c.page_sh) + (slot & ((int64_t(1) << a.c.page_sh) - 1));
    for (int w = 0; w < 2; ++w) {
      const float s = kv8_scale((w ? a.c.Vs : a.c.Ks)[at >> a.c.block_sh]);
      float y[4];
      kv8_f32x4<TYPE>(*reinterpret_cast<const uint32_t*>((w ? a.c.V : a.c.K) + at * D + d), y);
      *reinterpret_cast<uint2*>((w ? a.v_out : a.k_out) + row * D + d) =
          make_uint2(cvt_bf2(y[0] * s, y[1] * s), cvt_bf2(y[2] * s, y[3] * s));
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
  const int64_t blocks = std::min<int64_t>((T * Hkv * 2 + 3) / 4, 1 << 20);
#define EZ_GO(DD, TY) hipLaunchKernelGGL((ez::kv_quant_kernel<DD, TY>), dim3(unsigned(blocks)), dim3(256), 0, stream, a)
  EZ_KV8_DISPATCH(EZ_GO);
#undef EZ_GO
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
  const int64_t blocks = std::min<int64_t>((T * Hkv * (D / 4) + 255) / 256, 1 << 20);
#define EZ_GO(DD, TY) hipLaunchKernelGGL((ez::kv_dequant_kernel<DD, TY>), dim3(unsigned(blocks)), dim3(256), 0, stream, a)
  EZ_KV8_DISPATCH(EZ_GO);
#undef EZ_GO
  return ez::launch_status(op);
}
