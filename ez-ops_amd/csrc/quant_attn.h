// Arguments and checks that the kernels of attention over the 8-bit cache share.
#pragma once

#include <array>

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

inline int check_attn8(const char* op, const QuantAttnArgs& a, int64_t page_size, int64_t block, int64_t H, int64_t max_kv_len) {
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
