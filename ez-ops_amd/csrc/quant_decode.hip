// Attention over the 8-bit KV cache: one token per sequence (decode) and packed
// prompts or chunks, causal (prefill).
//
//   s_j = scale * q . (kc_j 2^(ek - 127)),  o = sum_j softmax(s)_j vc_j 2^(ev - 127)
//
// over the rows j that the query sees, in fp32.
#include "common.h"
#include "internal.h"
#include "quant_attn.h"
#include "prof.h"
#include "status.h"
#include "../../include/ezops_hip.h"

namespace ez {

EZ_PROF_DEFINE(quantdecode)
namespace {

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

}  // namespace
}  // namespace ez

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
  EZ_REQUIRE(B * H < int64_t(1) << 24, "%s: batch * heads past one launch", op);
  ez::finish_args(a, page_size, max_kv_len);
#define EZ_GO(DD, TY) hipLaunchKernelGGL((ez::quant_decode_kernel<DD, TY>), dim3(unsigned(B * H)), dim3(256), 0, stream, a)
  EZ_KV8_DISPATCH(EZ_GO);
#undef EZ_GO
  return ez::launch_status(op);
}
