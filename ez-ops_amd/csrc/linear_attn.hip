// Linear attention with a decay per head over packed ragged prompts, and its
// recurrent form for one token per sequence.
//
//   S_t = lambda S_{t-1} + k_t v_t^T          S [D, D] fp32 per (state slot, kv head)
//   o_t = scale * q_t^T S_t                   lambda = exp(log_decay[kv head])
//
// Query head h reads the state of kv head h / (H / Hkv).  lambda = 0 (log_decay
// -inf) is allowed: only powers lambda^n with n >= 0 appear, and lambda^0 = 1.
//
// A sequence's state lives in a pool of slots.  A sequence whose slot lies
// outside the pool, or that an earlier sequence of the batch holds already, is
// left out whole: nothing of it is read or written, so equal slots make no race.
#include "common.h"
#include "internal.h"
#include "prof.h"
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
  int B, H, Hkv;
  float scale;
};

// Slot of sequence b, -1 if it has none: outside the pool, or held by an earlier
// sequence.  Every thread of the block calls it (barrier inside).
template <int THREADS>
__device__ __forceinline__ int slot_of(const LinAttnArgs& a, int b) {
  const int s = a.state_slots ? a.state_slots[b] : b;
  int dup = 0;
  if (a.state_slots) {
    for (int c = threadIdx.x; c < b; c += THREADS) dup |= a.state_slots[c] == s;
    dup = __syncthreads_or(dup);
  }
  return s < 0 || s >= a.num_slots || dup ? -1 : s;
}

// One block per (sequence, kv head), thread = column of v: its column of the state
// in D registers, token by token.
template <int D>
__global__ __launch_bounds__(D) void linear_attn_prefill_kernel(LinAttnArgs a) {
  EZ_PROF_WAVE(kProfLinAttnPrefill);
  __shared__ float ks[D], qs[16][D];
  const int b = blockIdx.x / a.Hkv, kvh = blockIdx.x % a.Hkv, tid = threadIdx.x, G = a.H / a.Hkv;
  const int64_t t0 = min(max(int64_t(a.cu[b]), int64_t(0)), a.T);
  const int64_t t1 = min(min(int64_t(a.cu[b + 1]), a.T), t0 + a.max_q);
  int slot = -1;
  if (a.state) {
    slot = slot_of<D>(a, b);
    if (slot < 0) return;
  }
  if (t0 >= t1) return;
  float* st = a.state ? a.state + (int64_t(slot) * a.Hkv + kvh) * D * D + tid : nullptr;
  const bool cont = st && a.past && a.past[b] > 0;
  const float lambda = __expf(a.log_decay[kvh]);
  float S[D];
#pragma unroll
  for (int i = 0; i < D; ++i) S[i] = cont ? st[i * D] : 0.f;
  for (int64_t t = t0; t < t1; ++t) {
    __syncthreads();
    ks[tid] = bf2f(a.k[t * a.k_rs + kvh * D + tid]);
    for (int g = 0; g < G; ++g) qs[g][tid] = bf2f(a.q[t * a.q_rs + (kvh * G + g) * D + tid]);
    const float v = bf2f(a.v[t * a.v_rs + kvh * D + tid]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < D; ++i) S[i] = lambda * S[i] + ks[i] * v;
    for (int g = 0; g < G; ++g) {
      float o = 0.f;
#pragma unroll
      for (int i = 0; i < D; ++i) o += qs[g][i] * S[i];
      a.out[(t * a.H + kvh * G + g) * D + tid] = f2bf(o * a.scale);
    }
  }
  if (st) {
#pragma unroll
    for (int i = 0; i < D; ++i) st[i * D] = S[i];
  }
}

// One token per sequence: block = (sequence, kv head, slice of VC columns of the
// state), the slice in registers between its one read and its one write.
template <int D, int VC>
__global__ __launch_bounds__(256) void linear_attn_decode_kernel(LinAttnArgs a) {
  EZ_PROF_WAVE(kProfLinAttnDecode);
  constexpr int LPR = VC / 4;        // lanes per state row, 4 columns each
  constexpr int RPI = 256 / LPR;     // rows per step of the block
  constexpr int NI = D / RPI;        // rows per thread
  constexpr int NS = D / VC;
  __shared__ float ks[D], qs[16][D];
  __shared__ float4 red[RPI][LPR];
  const int tid = threadIdx.x, c = tid % LPR, r0 = tid / LPR, G = a.H / a.Hkv;
  const int sl = blockIdx.x % NS, kvh = blockIdx.x / NS % a.Hkv, b = blockIdx.x / NS / a.Hkv;
  const int slot = slot_of<256>(a, b);
  if (slot < 0) return;
  float4* st = reinterpret_cast<float4*>(a.state + (int64_t(slot) * a.Hkv + kvh) * D * D + sl * VC) + c;
  float4 S[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) S[i] = st[(r0 + i * RPI) * (D / 4)];
  const float lambda = __expf(a.log_decay[kvh]);
  for (int i = tid; i < D; i += 256) ks[i] = bf2f(a.k[b * a.k_rs + kvh * D + i]);
  for (int i = tid; i < G * D; i += 256) qs[i / D][i % D] = bf2f(a.q[b * a.q_rs + kvh * G * D + i]) * a.scale;
  const uint2 vr = *reinterpret_cast<const uint2*>(a.v + b * a.v_rs + kvh * D + sl * VC + 4 * c);
  const float4 v = make_float4(bf_lo(vr.x), bf_hi(vr.x), bf_lo(vr.y), bf_hi(vr.y));
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const float kk = ks[r0 + i * RPI];
    S[i].x = lambda * S[i].x + kk * v.x;
    S[i].y = lambda * S[i].y + kk * v.y;
    S[i].z = lambda * S[i].z + kk * v.z;
    S[i].w = lambda * S[i].w + kk * v.w;
    st[(r0 + i * RPI) * (D / 4)] = S[i];
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
    if (tid < VC) {
      float sum = 0.f;
      for (int r = 0; r < RPI; ++r) sum += reinterpret_cast<const float*>(&red[r][0])[tid];
      a.out[(int64_t(b) * a.H + kvh * G + g) * D + sl * VC + tid] = f2bf(sum);
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_common(const LinAttnArgs& a, int64_t H, int64_t Hkv, int64_t D, const char* what) {
  EZ_REQUIRE(a.q && a.k && a.v && a.log_decay && a.out, "%s: null pointer", what);
  EZ_REQUIRE(Hkv >= 1 && H >= 1 && H <= 4096 && H % Hkv == 0, "%s: num_heads must be divisible by num_kv_heads", what);
  const int64_t G = H / Hkv;
  EZ_REQUIRE(G == 1 || G == 2 || G == 4 || G == 8 || G == 16, "%s: group size %d not supported (1, 2, 4, 8 or 16)", what,
             int(G));
  EZ_REQUIRE(D == 64 || D == 128, "%s: head_dim must be 64 or 128", what);
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
  return 0;
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
  const int rc = ez::check_common(a, H, Hkv, D, "linear_attn_prefill");
  if (rc != EZ_OK) return rc;
  EZ_REQUIRE(cu_seqlens, "linear_attn_prefill: null pointer");
  EZ_REQUIRE(B >= 1 && B <= 65536 && T >= 1 && T < (int64_t(1) << 30),
             "linear_attn_prefill: batch must be in [1, 65536] and tokens in [1, 2^30)");
  EZ_REQUIRE(!state || (num_slots >= 1 && num_slots < (int64_t(1) << 31)),
             "linear_attn_prefill: num_slots must be in [1, 2^31)");
  EZ_REQUIRE(max_q_len >= 0, "linear_attn_prefill: max_q_len must be >= 0");
  a.B = int(B); a.H = int(H); a.Hkv = int(Hkv);
  a.scale = scale > 0.f ? scale : 1.f / sqrtf(float(D));
  if (D == 64) hipLaunchKernelGGL(ez::linear_attn_prefill_kernel<64>, dim3(unsigned(B * Hkv)), dim3(64), 0, stream, a);
  else hipLaunchKernelGGL(ez::linear_attn_prefill_kernel<128>, dim3(unsigned(B * Hkv)), dim3(128), 0, stream, a);
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
  const int rc = ez::check_common(a, H, Hkv, D, "linear_attn_decode");
  if (rc != EZ_OK) return rc;
  EZ_REQUIRE(state, "linear_attn_decode: null pointer");
  EZ_REQUIRE(B >= 1 && B <= 65536, "linear_attn_decode: batch must be in [1, 65536]");
  EZ_REQUIRE(num_slots >= 1 && num_slots < (int64_t(1) << 31), "linear_attn_decode: num_slots must be in [1, 2^31)");
  a.B = int(B); a.H = int(H); a.Hkv = int(Hkv);
  a.scale = scale > 0.f ? scale : 1.f / sqrtf(float(D));
  const dim3 grid(unsigned(B * Hkv));
  if (D == 64) hipLaunchKernelGGL((ez::linear_attn_decode_kernel<64, 64>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((ez::linear_attn_decode_kernel<128, 128>), grid, dim3(256), 0, stream, a);
  return ez::launch_status("linear_attn_decode");
}
