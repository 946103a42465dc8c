// Attention over the 8-bit KV cache: one token per sequence (decode) and packed
// prompts or chunks, causal (prefill).
//
//   s_j = scale * q . (kc_j 2^(ek - 127)),  o = sum_j softmax(s)_j vc_j 2^(ev - 127)
//
// over the rows j that the query sees, in fp32.
#include "common.h"
#include "internal.h"
#include "kv8.h"
#include "prof.h"
#include "status.h"
#include "../../include/ezops_hip.h"

namespace ez {

EZ_PROF_DEFINE(quantattn)
namespace {

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

__device__ __forceinline__ int64_t cache_at(const QuantAttnArgs& a, int64_t b, int h, int64_t row) {
  const uint32_t id = min(uint32_t(a.table[b * a.M + (row >> a.c.page_sh)]), uint32_t(a.c.num_pages - 1));
  return ((int64_t(id) * a.c.Hkv + h) << a.c.page_sh) + (row & ((int64_t(1) << a.c.page_sh) - 1));
}

// One block per (query row, head): its waves take every fourth cache row.
template <int D, int TYPE>
__device__ void attend(const QuantAttnArgs& a, int64_t b, int64_t t, int hq, int64_t L) {
  constexpr int E = D / kWave;
  __shared__ float Os[4][D], Ms[4], Ls[4];
  const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x >> 6;
  const int h = hq / (a.H / a.c.Hkv);
  float q[E], o[E] = {}, m = -INFINITY, l = 0.f;
  for (int e = 0; e < E; ++e) q[e] = bf2f(a.q[t * a.q_rs + int64_t(hq) * D + lane * E + e]);
  for (int64_t j = w; j < L; j += 4) {
    const int64_t at = cache_at(a, b, h, j);
    float k[4], v[4], s = 0.f;
    uint32_t kw = 0, vw = 0;
    for (int e = 0; e < E; ++e) {
      kw |= uint32_t(a.c.K[at * D + lane * E + e]) << (8 * e);
      vw |= uint32_t(a.c.V[at * D + lane * E + e]) << (8 * e);
    }
    kv8_f32x4<TYPE>(kw, k);
    kv8_f32x4<TYPE>(vw, v);
    for (int e = 0; e < E; ++e) s += q[e] * k[e];
    s = wave_sum(s) * kv8_scale(a.c.Ks[at >> a.c.block_sh]) * a.scale;
    const float mn = fmaxf(m, s), al = m == -INFINITY ? 0.f : expf(m - mn), p = expf(s - mn);
    const float vs = kv8_scale(a.c.Vs[at >> a.c.block_sh]);
    l = l * al + p;
    for (int e = 0; e < E; ++e) o[e] = o[e] * al + p * vs * v[e];
    m = mn;
  }
  for (int e = 0; e < E; ++e) Os[w][lane * E + e] = o[e];
  if (lane == 0) {
    Ms[w] = m;
    Ls[w] = l;
  }
  __syncthreads();
  if (threadIdx.x < D) {
    const float M = fmaxf(fmaxf(Ms[0], Ms[1]), fmaxf(Ms[2], Ms[3]));
    float ov = 0.f, lv = 0.f;
    for (int i = 0; i < 4; ++i) {
      const float f = Ms[i] == -INFINITY && Ls[i] == 0.f ? 0.f : expf(Ms[i] - M);
      ov += f * Os[i][threadIdx.x];
      lv += f * Ls[i];
    }
    a.out[(t * a.H + hq) * D + threadIdx.x] = f2bf(L > 0 ? ov / lv : 0.f);
  }
}

template <int D, int TYPE>
__global__ __launch_bounds__(256) void quant_decode_kernel(QuantAttnArgs a) {
  EZ_PROF_WAVE(kProfQuantAttnDecode);
  const int64_t b = blockIdx.x / a.H;
  attend<D, TYPE>(a, b, b, int(blockIdx.x % a.H), min(max(int64_t(a.kv_lens[b]), int64_t(0)), a.cap));
}

template <int D, int TYPE>
__global__ __launch_bounds__(256) void quant_prefill_kernel(QuantAttnArgs a) {
  EZ_PROF_WAVE(kProfQuantAttnPrefill);
  const int64_t t = blockIdx.x / a.H;
  for (int64_t b = 0; b < a.B; ++b) {
    const int64_t r0 = max(int64_t(a.cu[b]), int64_t(0)), r1 = min(int64_t(a.cu[b + 1]), a.T);
    if (t < r0 || t >= r1) continue;
    const int64_t past = a.past ? max(int64_t(a.past[b]), int64_t(0)) : 0;
    const int64_t pos = past + t - r0;
    if (pos < a.cap) attend<D, TYPE>(a, b, t, int(blockIdx.x % a.H), pos + 1);
    return;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_attn8(const char* op, const QuantAttnArgs& a, int64_t page_size, int64_t block, int64_t H, int64_t max_kv_len) {
  EZ_REQUIRE(a.q && a.out && a.table, "%s: null pointer", op);
  const int rc = check_kv8(op, a.c, page_size, block);
  if (rc != EZ_OK) return rc;
  EZ_REQUIRE(a.B >= 1 && a.B <= 65536, "%s: batch must be in [1, 65536]", op);
  EZ_REQUIRE(a.T >= 1 && a.T < (int64_t(1) << 30), "%s: tokens must be in [1, 2^30)", op);
  const int64_t Hkv = a.c.Hkv;
  EZ_REQUIRE(H >= 1 && Hkv >= 1 && H <= 4096 && H % Hkv == 0,
             "%s: num_heads must be in [1, 4096] and divisible by num_kv_heads", op);
  const int64_t G = H / Hkv;
  EZ_REQUIRE(G == 1 || G == 2 || G == 4 || G == 8 || G == 16, "%s: group size must be 1, 2, 4, 8 or 16", op);
  EZ_REQUIRE(a.c.D == 64 || a.c.D == 128, "%s: head_dim must be 64 or 128", op);
  EZ_REQUIRE(a.M >= 1 && a.M * page_size <= (int64_t(1) << 30),
             "%s: max_pages must be >= 1 and max_pages * page_size at most 2^30", op);
  EZ_REQUIRE(max_kv_len >= 0, "%s: max_kv_len must be >= 0", op);
  EZ_REQUIRE(a.q_rs >= H * a.c.D, "%s: token strides below the heads' size", op);
  EZ_REQUIRE(a.q_rs % 8 == 0 && aligned16(a.q) && aligned16(a.out), "%s: rows of q and out must begin at multiples of 16 bytes",
             op);
  EZ_REQUIRE(a.scale < INFINITY, "%s: scale must be finite", op);
  const int64_t pool = kv8_pool_bytes(a.c), sc = kv8_scale_bytes(a.c), no = a.T * H * a.c.D * 2;
  const struct { const void* p; int64_t n; } in[] = {
      {a.c.K, pool}, {a.c.V, pool}, {a.c.Ks, sc}, {a.c.Vs, sc}, {a.table, a.B * a.M * 4}, {a.kv_lens, a.B * 4},
      {a.cu, (a.B + 1) * 4}, {a.past, a.B * 4}, {a.q, ((a.T - 1) * a.q_rs + H * a.c.D) * 2}};
  for (const auto& x : in) EZ_REQUIRE(!overlap(a.out, no, x.p, x.n), "%s: out overlaps an input", op);
  EZ_REQUIRE(a.T * H < int64_t(1) << 24, "%s: tokens * heads past one launch", op);
  return EZ_OK;
}

void finish_args(QuantAttnArgs& a, int64_t page_size, int64_t max_kv_len) {
  a.cap = a.M * page_size;
  if (max_kv_len > 0 && max_kv_len < a.cap) a.cap = max_kv_len;
  if (!(a.scale > 0.f)) a.scale = 1.f / sqrtf(float(a.c.D));
}

}  // namespace
}  // namespace ez

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

extern "C" size_t ezops_quant_paged_attn_decode_workspace_size(int64_t B, int64_t H, int64_t Hkv, int64_t D,
                                                               int64_t kv_len) {
  return 0;
}

extern "C" int ezops_quant_paged_attn_decode_bf16(const void* q, int64_t q_stride, const void* K_cache, const void* V_cache,
                                                  const void* K_scale, const void* V_scale, int cache_type,
                                                  const int32_t* block_table, const int32_t* kv_lens, void* out, int64_t B,
                                                  int64_t H, int64_t Hkv, int64_t D, int64_t num_pages, int64_t page_size,
                                                  int64_t max_pages, int64_t block_size, int64_t max_kv_len, float scale,
                                                  void* ws, size_t ws_bytes, hipStream_t stream) {
  const char* op = "quant_paged_attn_decode";
  ez::QuantAttnArgs a{};
  ez::fill_kv8(a.c, K_cache, V_cache, K_scale, V_scale, cache_type, num_pages, page_size, block_size, Hkv, D);
  a.q = static_cast<const uint16_t*>(q); a.q_rs = q_stride;
  a.out = static_cast<uint16_t*>(out);
  a.table = block_table; a.kv_lens = kv_lens;
  a.B = a.T = B; a.M = max_pages; a.H = int(H); a.scale = scale;
  EZ_REQUIRE(kv_lens, "%s: null pointer", op);
  const int rc = ez::check_attn8(op, a, page_size, block_size, H, max_kv_len);
  if (rc != EZ_OK) return rc;
  ez::finish_args(a, page_size, max_kv_len);
#define EZ_GO(DD, TY) hipLaunchKernelGGL((ez::quant_decode_kernel<DD, TY>), dim3(unsigned(B * H)), dim3(256), 0, stream, a)
  EZ_KV8_DISPATCH(EZ_GO);
#undef EZ_GO
  return ez::launch_status(op);
}

extern "C" size_t ezops_quant_prefill_attn_workspace_size(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t D,
                                                          int64_t max_kv_len) {
  return 0;
}

extern "C" int ezops_quant_prefill_attn_bf16(const void* q, int64_t q_stride, const void* K_cache, const void* V_cache,
                                             const void* K_scale, const void* V_scale, int cache_type,
                                             const int32_t* block_table, const int32_t* cu_seqlens, const int32_t* past_lens,
                                             void* out, int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t D,
                                             int64_t num_pages, int64_t page_size, int64_t max_pages, int64_t block_size,
                                             int64_t max_kv_len, float scale, void* ws, size_t ws_bytes,
                                             hipStream_t stream) {
  const char* op = "quant_prefill_attn";
  ez::QuantAttnArgs a{};
  ez::fill_kv8(a.c, K_cache, V_cache, K_scale, V_scale, cache_type, num_pages, page_size, block_size, Hkv, D);
  a.q = static_cast<const uint16_t*>(q); a.q_rs = q_stride;
  a.out = static_cast<uint16_t*>(out);
  a.table = block_table; a.cu = cu_seqlens; a.past = past_lens;
  a.B = B; a.T = T; a.M = max_pages; a.H = int(H); a.scale = scale;
  EZ_REQUIRE(cu_seqlens, "%s: null pointer", op);
  const int rc = ez::check_attn8(op, a, page_size, block_size, H, max_kv_len);
  if (rc != EZ_OK) return rc;
  ez::finish_args(a, page_size, max_kv_len);
#define EZ_GO(DD, TY) hipLaunchKernelGGL((ez::quant_prefill_kernel<DD, TY>), dim3(unsigned(T * H)), dim3(256), 0, stream, a)
  EZ_KV8_DISPATCH(EZ_GO);
#undef EZ_GO
  return ez::launch_status(op);
}
