// Causal attention of packed prompts and chunks over the 8-bit KV cache.
//
//   s_j = scale * q . kc_j 2^(ek - 127),  o = sum_j softmax(s)_j vc_j 2^(ev - 127)
//
// kc, vc are the codes, ek, ev the exponents of the key's block of rows (at least 16
// rows each).  Both products run on v_mfma_f32_32x32x16_bf16 with the codes as they are
// (int8 and e4m3 are exact in bf16), and the scales enter the softmax, whose weights
// are taken in the exp2 domain: with c = scale log2(e) 2^(ek - 127) and v = ev - 127
//
//   w_j = 2^(c s'_j - m + v)   s' = q . kc      (the weight times the scale of v)
//   o  += w_j vc_j,  l += w_j 2^-v
//
// so a scale costs nothing per key: c and v - m are the operands of the fused
// multiply-add that the exponent needs anyway, 2^-v the other factor of the dot product
// that sums the weights.  w is rounded to bf16 for the product; l sums the rounded
// weights, so that rounding cancels in o / l but for its spread.
//
// A block owns 256 rows of one kv head (128 with heads of 64): (query, head of the group)
// pairs, 256 / G queries, 32 rows to each of 8 (4) waves; all share the K / V tiles of 64
// keys.  A tile is read once from memory in 8 bits (16 bytes a thread and tensor, two tiles
// ahead in registers), widened to bf16 on its way into one of two LDS buffers, so the
// widening is done once for all waves.  Operand layouts (lane 32 h + j): S^T = K Q^T, then O^T = V^T P^T
// with the weights staying in their lane; V^T by transposing LDS reads.
//
// Where the queries are few (a chunk on a long prefix) the keys are shared out over
// nsplit blocks; they leave fp32 partials (O, m, l), which a second kernel joins.
//
// Measured (two cards): 2048 tokens on 30000 rows, 32 / 8 heads of 128, e4m3: 1.03 and 1.08 ms,
// 1010 and 970 TFLOP/s; a fresh prompt of 4096 tokens, int8: 145 and 153 us, 950 and 900 (a large
// bf16 matrix product: 1220).  By the counters the matrix cores are busy 44% and the vector units
// 51% of a CU's time at 4096 tokens, hardly at once: a tile's exponentials take as long as its
// products, the two waves of a SIMD meet at each tile's barrier, and a second tile's scores do
// not fit the registers (228 of 256).  8192 tokens of 16 / 2 heads of 64: 204 us, 670 TFLOP/s;
// with as many exponentials for half the products the vector units are busy 76% of the time,
// the matrix cores 34%.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "internal.h"
#include "prof.h"
#include "quant_attn.h"
#include "status.h"
#include "../../include/ezops_hip.h"

namespace ez {

EZ_PROF_DEFINE(quantprefill)
namespace {

constexpr float kLazy = 8.f;     // log2 headroom of the softmax reference, see below
// Waves of a block, 32 (query, head) rows each.
constexpr int waves_of(int64_t D) { return D == 64 ? 4 : 8; }
constexpr int rows_of(int64_t D) { return 32 * waves_of(D); }
constexpr int kBK = 64;          // keys of a tile
constexpr int kMaxSplits = 32;
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

struct SplitPlan {
  int nsplit;
  int tiles;   // query tiles of all sequences, at most
  float* o;    // partials [nsplit][T * H][D]
  float* ml;   // [nsplit][T * H][2]
};

__device__ __forceinline__ float halves_max(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// A query tile: QT queries from query `first` on of the sequence whose rows begin at t0.
struct QueryTile {
  int b, t0, qlen, past, first;
};

// The idx-th query tile of the batch; false if there are fewer.  A sequence's last tiles,
// which see the most keys, come first.  Offsets and lengths come from the device and may
// hold anything: they are clamped into the rows and the cache.
template <int QT>
__device__ __forceinline__ bool find_tile(const QuantAttnArgs& a, int idx, QueryTile& q) {
  const int lane = threadIdx.x & (kWave - 1), T = int(a.T), cap = int(a.cap);
  const int B = int(a.B);
  int c0 = 0, c1 = 0, p0 = 0;  // of sequence b0 + lane, read a step ahead
  auto ask = [&](int b) {
    b = min(b, B - 1);
    c0 = a.cu[b];
    c1 = a.cu[b + 1];
    p0 = a.past ? a.past[b] : 0;
  };
  ask(lane);
  for (int b0 = 0; b0 < B; b0 += kWave) {
    const int t0 = min(max(c0, 0), T), past = min(max(p0, 0), cap);
    const int n = b0 + lane < B ? min(min(max(c1, 0), T) - t0, cap - past) : 0;
    ask(b0 + kWave + lane);
    const int tiles = n > 0 ? (n + QT - 1) / QT : 0;
    const int end = wave_scan(tiles);
    const uint64_t hit = __ballot(idx < end);
    if (hit) {
      const int l = __ffsll(static_cast<unsigned long long>(hit)) - 1;
      q.b = b0 + l;
      q.t0 = __builtin_amdgcn_readlane(t0, l);
      q.qlen = __builtin_amdgcn_readlane(n, l);
      q.past = __builtin_amdgcn_readlane(past, l);
      q.first = (__builtin_amdgcn_readlane(end, l) - 1 - idx) * QT;
      return true;
    }
    idx -= __builtin_amdgcn_readlane(end, kWave - 1);
  }
  return false;
}

// Key tiles of a split of the tile's `n` key tiles; splits behind the last one with any leave.
// The host plans with a bound on the lengths that may be far above them: three tiles at least
// (70 tokens on 3000 rows planned for 131072: 37 us with 32 splits, two tiles each).
constexpr int kMinTiles = 3;
__device__ __forceinline__ int split_tiles(int n, int nsplit) { return max((n + nsplit - 1) / nsplit, kMinTiles); }

__device__ __forceinline__ bool has_nan_code(uint32_t w) {  // an e4m3 byte of 0x7f or 0xff
  const uint32_t x = (w & 0x7f7f7f7fu) ^ 0x7f7f7f7fu;
  return ((x - 0x01010101u) & ~x & 0x80808080u) != 0;
}
__device__ __forceinline__ uint32_t without_nan(uint32_t w) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (((w >> (8 * i)) & 0x7f) == 0x7f) w &= ~(0xffu << (8 * i));
  return w;
}

template <int D, int TYPE, int G>
__global__ __launch_bounds__(waves_of(D) * kWave) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2))) void quant_prefill_kernel(QuantAttnArgs a,
                                                                                                          SplitPlan pl) {
  EZ_PROF_WAVE(kProfQuantAttnPrefill);
  constexpr int QT = rows_of(D) / G;  // queries of a block
  constexpr int NS = D / 16;        // 16-dim steps of S
  constexpr int ND = D / 32;        // 32-dim blocks of O^T
  constexpr int CPR = D / 8;        // 16-byte chunks of a bf16 row in LDS
  constexpr int TPR = D / 16;       // threads that stage a row
  static_assert(kBK * TPR == waves_of(D) * kWave, "a thread stages 16 bytes of K and of V");
  __shared__ __align__(16) uint16_t Ks[2][kBK * D];  // [key][chunk ^ key % CPR]
  __shared__ __align__(16) uint16_t Vs[2][kBK * D];  // [key][chunk ^ vswz(key)]
  __shared__ __align__(16) float Cs[2][12];          // of each 16 keys: c, v, 2^-v twice in bf16
  __shared__ int nan_tile[2];                        // first key of the tile whose NaN codes of V were taken out

  const int kvh = int(blockIdx.x % unsigned(a.c.Hkv));
  const int rest = int(blockIdx.x / unsigned(a.c.Hkv));
  const int split = rest % pl.nsplit;
  QueryTile qt;
  if (!find_tile<QT>(a, rest / pl.nsplit, qt)) return;
  const int kend = qt.past + min(qt.qlen, qt.first + QT);  // keys [0, kend) serve this block
  const int ntiles = (kend + kBK - 1) / kBK, per = split_tiles(ntiles, pl.nsplit);
  const int tile0 = split * per, n = min(per, ntiles - tile0);
  if (n <= 0) return;

  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, j = lane & 31;
  const int row = wave * 32 + j;
  const int qi = min(qt.first + row / G, qt.qlen - 1);  // rows past the sequence compute, never store
  const bool live = qt.first + row / G < qt.qlen;
  const int hq = kvh * G + row % G;
  const int qpos = qt.past + qi;
  const int wave_q0 = qt.first + wave * 32 / G;
  const bool wave_on = wave_q0 < qt.qlen;
  const int wave_first = qt.past + wave_q0, wave_last = qt.past + min(qt.first + (wave * 32 + 31) / G, qt.qlen - 1);

  bf16x8_t qf[NS];
  {
    const uint16_t* qp = a.q + int64_t(qt.t0 + qi) * a.q_rs + int64_t(hq) * D + 8 * h;
#pragma unroll
    for (int s = 0; s < NS; ++s) qf[s] = as_bf16x8(*reinterpret_cast<const uint4*>(qp + 16 * s));
  }

  // ---- staging: thread = (key sr of the tile, 16 dims from 16 sc on)
  const int sr = tid / TPR, sc = tid % TPR;
  const bool stage_c = sr % 16 == 0 && sc == 0;
  const int32_t* table = a.table + int64_t(qt.b) * a.M;
  const int pmask = (1 << a.c.page_sh) - 1;
  auto key_row = [&](int t) { return min((tile0 + t) * kBK + sr, kend - 1); };
  auto flat_row = [&](int r, int32_t id) {
    const uint32_t page = min(uint32_t(id), uint32_t(a.c.num_pages - 1));
    return ((int64_t(page) * a.c.Hkv + kvh) << a.c.page_sh) + (r & pmask);
  };
  // Two tiles are in flight in registers, the tile of parity P in slot P; the page of a tile is
  // asked for two tiles before its codes, ahead of theirs, so that no wait for it waits for them.
  uint4 raw[2][2];  // [parity][K, V]
  int ek[2] = {0, 0}, ev[2] = {0, 0};
  auto page_of = [&](int t) { return table[key_row(t) >> a.c.page_sh]; };
  int32_t id[2] = {page_of(0), page_of(1)};
  auto issue = [&](int t, auto parity) {  // tile t's codes and exponents
    constexpr int P = decltype(parity)::value;
    const int64_t at = flat_row(key_row(t), id[P]);
    id[P] = page_of(t + 2);
    raw[P][0] = *reinterpret_cast<const uint4*>(a.c.K + at * D + 16 * sc);
    raw[P][1] = *reinterpret_cast<const uint4*>(a.c.V + at * D + 16 * sc);
    if (stage_c) {
      ek[P] = a.c.Ks[at >> a.c.block_sh];
      ev[P] = a.c.Vs[at >> a.c.block_sh];
    }
  };
  auto vswz = [](int r) { return D == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); };
  auto put = [&](uint16_t* dst, int swz, const uint4& v) {
    const uint2 p0 = kv8_bf16x4<TYPE>(v.x), p1 = kv8_bf16x4<TYPE>(v.y), p2 = kv8_bf16x4<TYPE>(v.z), p3 = kv8_bf16x4<TYPE>(v.w);
    *reinterpret_cast<uint4*>(dst + sr * D + ((2 * sc) ^ swz) * 8) = make_uint4(p0.x, p0.y, p1.x, p1.y);
    *reinterpret_cast<uint4*>(dst + sr * D + ((2 * sc + 1) ^ swz) * 8) = make_uint4(p2.x, p2.y, p3.x, p3.y);
  };
  auto stage = [&](int t, auto parity) {  // tile t from its registers into its buffer
    constexpr int buf = decltype(parity)::value;
    const int k0 = (tile0 + t) * kBK;
    if (TYPE == kKvE4m3 && k0 + kBK - 1 > qt.past + qt.first) {
      // Some query of the block does not see some key of the tile: its weight of 0 must not
      // meet a NaN.  The codes go, and fix_nan puts them back where they are seen.
      uint4& v = raw[buf][1];
      if (has_nan_code(v.x) || has_nan_code(v.y) || has_nan_code(v.z) || has_nan_code(v.w)) {
        v = make_uint4(without_nan(v.x), without_nan(v.y), without_nan(v.z), without_nan(v.w));
        nan_tile[buf] = k0;
      }
    }
    put(Ks[buf], sr % CPR, raw[buf][0]);
    put(Vs[buf], vswz(sr), raw[buf][1]);
    if (stage_c) {
      const int k = kv8_exp(ek[buf]), v = kv8_exp(ev[buf]), u = sr / 16;
      const bool nan = v == kKvNanExp;
      Cs[buf][u] = kv8_factor(a.scale, k);
      Cs[buf][4 + u] = nan ? __uint_as_float(0x7fc00000u) : float(v - 127);
      Cs[buf][8 + u] = __uint_as_float(nan ? 0x3f803f80u : uint32_t(254 - v) << 7 | uint32_t(254 - v) << 23);
    }
  };
  if (tid < 2) nan_tile[tid] = -1;
  __syncthreads();
  using even = std::integral_constant<int, 0>;
  using odd = std::integral_constant<int, 1>;
  issue(0, even{});
  if (n > 1) issue(1, odd{});
  stage(0, even{});
  if (n > 2) issue(2, even{});
  __syncthreads();

  // ---- operand addresses: K row 32 kk + j has the swizzle of row j; lane (i = 16 g1 + mm,
  // half h) of the transposing reads takes key 4 h + mm / 4 (+ 8, + 16-key step), dims
  // 32 d + 16 g1 + 4 (mm % 4) .. + 3.
  int koff[NS], voff[ND];
#pragma unroll
  for (int s = 0; s < NS; ++s) koff[s] = j * D + ((2 * s + h) ^ (j % CPR)) * 8;
  {
    const int mm = lane & 15, g1 = (lane >> 4) & 1, vrow = 4 * h + (mm >> 2);
#pragma unroll
    for (int d = 0; d < ND; ++d)
      voff[d] = vrow * D + ((4 * d + 2 * g1 + ((mm & 3) >> 1)) ^ vswz(vrow)) * 8 + (mm & 1) * 4;
  }

  f32x16_t o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m = kLowest, l = 0.f;

  auto compute = [&](int t, auto parity) {
    constexpr int buf = decltype(parity)::value;
    const int k0 = (tile0 + t) * kBK;
    const bool edge = k0 + kBK - 1 > wave_first;  // some of the wave's queries do not see all of the tile
    const uint16_t* ks = Ks[buf];
    f32x16_t st[2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int r = 0; r < 16; ++r) st[kk][r] = 0.f;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int s = 0; s < NS; ++s)
        st[kk] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            as_bf16x8(*reinterpret_cast<const uint4*>(ks + 32 * kk * D + koff[s])), qf[s], st[kk], 0, 0, 0);
    // The reads run NS steps ahead of the products (left alone they run one ahead, and
    // every pair of products waits out the latency of LDS).
    __builtin_amdgcn_sched_group_barrier(0x100, NS, 0);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, NS, 0);
    // st[kk][r] = s' of (query j, key k0 + 32 kk + 8 (r / 4) + 4 h + r % 4); 16 keys u = 2 kk + r / 8 share a scale
    float c[4], v[4], iv[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      c[u] = Cs[buf][u];
      v[u] = Cs[buf][4 + u];
      iv[u] = Cs[buf][8 + u];
    }
    if (edge) {
      const int seen = qpos - k0;  // keys of the tile up to this one are seen
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // scales of keys that are not seen may be NaN
        c[u] = 16 * u > seen ? 1.f : c[u];
        v[u] = 16 * u > seen ? 0.f : v[u];
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * kk + 8 * (r >> 2) + (r & 3) > seen - 4 * h) st[kk][r] = -INFINITY;
    }
    float mx = kLowest;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float g = st[u >> 1][8 * (u & 1)];
#pragma unroll
      for (int r = 1; r < 8; ++r) g = fmaxf(g, st[u >> 1][8 * (u & 1) + r]);
      mx = fmaxf(mx, g * c[u]);
    }
    mx = halves_max(mx);
    // The reference m moves, and O and l are rescaled, only where a row's maximum passes
    // it by more than kLazy, and most tiles skip the rescale.  Weights, which carry the scale
    // of v, stay below 2^(kLazy + 60), and the sums of their products with codes far below
    // 2^127: fp32 and bf16 hold them with the same relative precision at any size.
    if (__builtin_amdgcn_ballot_w64(mx > m + kLazy)) {
      const float mn = fmaxf(m, mx);
      const float alpha = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= alpha;
    }
    const uint16_t* vs = Vs[buf];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      // 16 keys: slots 8 h .. 8 h + 7 of the product are registers 8 (u % 2) .. + 7
      uint32_t w[4];
      const float off = v[u] - m;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(st[u >> 1][8 * (u & 1) + 2 * q], c[u], off));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(st[u >> 1][8 * (u & 1) + 2 * q + 1], c[u], off));
        w[q] = cvt_bf2(p0, p1);
        l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w[q]), __builtin_bit_cast(bf16x2_t, iv[u]), l, false);
      }
      const bf16x8_t pb = as_bf16x8(make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const uint16_t* vp = vs + 16 * u * D + voff[d];
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)vp);
        const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(vp + 8 * D));
        const bf16x8_t va = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va, pb, o[d], 0, 0, 0);
      }
    }
    if (TYPE == kKvE4m3 && nan_tile[buf] == k0) {  // corrupt rows only: NaN where a query sees one
      for (int i = 0; i < kBK && k0 + i < kend; ++i) {
        const int r = k0 + i;
        const uint8_t* vr = a.c.V + flat_row(r, table[r >> a.c.page_sh]) * D + 4 * h;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t x = *reinterpret_cast<const uint32_t*>(vr + 32 * d + 8 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (r <= qpos && ((x >> (8 * e)) & 0x7f) == 0x7f) o[d][4 * q + e] = __uint_as_float(0x7fc00000u);
          }
      }
    }
  };

  auto step = [&](int t, auto parity, auto other) {
    if (t + 1 < n) {
      stage(t + 1, other);  // its buffer was read last before the barrier behind tile t - 1
      if (t + 3 < n) issue(t + 3, other);
    }
    if (wave_on && (tile0 + t) * kBK <= wave_last) compute(t, parity);
    __syncthreads();
  };
  for (int t = 0; t < n; t += 2) {
    step(t, even{}, odd{});
    if (t + 1 < n) step(t + 1, odd{}, even{});
  }

  // ---- l: the two lane halves hold a share of query j's sum each
  l = halves_sum(l);
  if (!live) return;
  if (pl.nsplit == 1) {
    const float inv = 1.f / l;
    uint16_t* op = a.out + (int64_t(qt.t0 + qi) * a.H + hq) * D + 4 * h;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q)  // o[d][4q + e] = O^T[dim 32d + 8q + 4h + e][row j]
        *reinterpret_cast<uint2*>(op + 32 * d + 8 * q) = make_uint2(cvt_bf2(o[d][4 * q] * inv, o[d][4 * q + 1] * inv),
                                                                    cvt_bf2(o[d][4 * q + 2] * inv, o[d][4 * q + 3] * inv));
  } else {
    const int64_t at = (int64_t(split) * a.T + qt.t0 + qi) * a.H + hq;
    float* op = pl.o + at * D + 4 * h;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<float4*>(op + 32 * d + 8 * q) =
            make_float4(o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]);
    if (h == 0) *reinterpret_cast<float2*>(pl.ml + at * 2) = make_float2(m, l);
  }
}

// Joins the splits of one query tile's rows of a kv head: 4 dims a thread.
template <int D, int G>
__global__ __launch_bounds__(256) void quant_prefill_join_kernel(QuantAttnArgs a, SplitPlan pl) {
  EZ_PROF_WAVE(kProfQuantAttnCombine);
  constexpr int QT = rows_of(D) / G, TPR = D / 4, PER = 256 / TPR;  // rows of a block
  constexpr int parts = rows_of(D) / PER;
  const int part = int(blockIdx.x) % parts, rest = int(blockIdx.x) / parts;
  const int kvh = rest % a.c.Hkv;
  QueryTile qt;
  if (!find_tile<QT>(a, rest / a.c.Hkv, qt)) return;
  const int row = part * PER + int(threadIdx.x) / TPR, d = int(threadIdx.x) % TPR * 4;
  const int qi = qt.first + row / G;
  if (qi >= qt.qlen) return;
  const int kend = qt.past + min(qt.qlen, qt.first + QT), ntiles = (kend + kBK - 1) / kBK;
  const int per = split_tiles(ntiles, pl.nsplit), used = (ntiles + per - 1) / per;
  const int64_t at = int64_t(qt.t0 + qi) * a.H + kvh * G + row % G, step = a.T * a.H;
  float o[4];
  if (pl.nsplit <= 4) join_parts<4>(reinterpret_cast<const float2*>(pl.ml) + at, reinterpret_cast<const float4*>(pl.o + at * D + d), step,
             step * (D / 4), used, o);
  else join_parts<16>(reinterpret_cast<const float2*>(pl.ml) + at, reinterpret_cast<const float4*>(pl.o + at * D + d), step,
             step * (D / 4), used, o);
  *reinterpret_cast<uint2*>(a.out + at * D + d) = make_uint2(cvt_bf2(o[0], o[1]), cvt_bf2(o[2], o[3]));
}

// Query tiles at most (a sequence adds at most one that is not full), and the splits of
// the keys that a model of the time prefers, in us: a block takes kBlock to begin and end and
// kTile a key tile; the kernel lasts as long as its longest block, as the blocks' sum over
// the CUs, and with several sequences, whose blocks come in no order of size, as whole rounds
// of them; splits add a join and their partials through memory.  The longest block has the
// key tiles of kv_len, a mean one those of the middle row of one prompt that ends there, or
// three quarters where there are several sequences (the lengths are on the device).  70
// tokens on 3000 rows of 32 / 8 heads: 6, 12, 16 and 24 splits take 32.7, 28.7, 28.7 and
// 37 us; 16 x 16 tokens on 2000 rows 56.8, 49.9 and 58 us with one, two and three; nine
// ragged chunks of 2660 tokens of 16 / 2 heads of 64 on up to 2500 rows 61 and 58 us with
// one and two.
//
// kv_len counts in steps of len_step, so that most_splits below sees every plan.
constexpr int64_t kMaxLen = int64_t(1) << 30;
int64_t len_step(int64_t n) {  // a sixteenth to an eighth of n, two key tiles at least
  return std::max(int64_t(2 * kBK), (int64_t(1) << (63 - __builtin_clzll(static_cast<unsigned long long>(n)))) / 8);
}
int64_t len_up(int64_t n) {
  n = std::min(n, kMaxLen);
  return (n + len_step(n) - 1) / len_step(n) * len_step(n);
}
int split_limit(int64_t kv_len) { return int(std::min(int64_t(kMaxSplits), (kv_len + 2 * kBK - 1) / (2 * kBK))); }
SplitPlan plan(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t kv_len) {
  kv_len = len_up(kv_len);
  const int64_t qt = rows_of(D) / (H / Hkv), seqs = B < T ? B : T;
  const int64_t tiles = (T + seqs * (qt - 1)) / qt;
  const double blocks = double(seqs * ((T / seqs + qt - 1) / qt) * Hkv), cus = num_cus();
  const double kTile = D == 64 ? 1.2 : 2.2, kBlock = 7.0, at_once = D == 64 ? 3.0 : 1.0;
  const double most = double(kv_len) / kBK + 1;
  const double mean = seqs > 1 ? most * 0.75 : kv_len > T ? double(kv_len - T / 2) / kBK : most / 2;
  int best = 1;
  double least = 1e30;
  for (int ns = 1; ns <= split_limit(kv_len); ++ns) {
    const double longest = most / ns * kTile + kBlock, sum = blocks * (mean * kTile + ns * kBlock / at_once) / cus;
    const double rounds = seqs > 1 ? std::ceil(blocks * ns / (cus * at_once)) : 1.0;
    const double whole = rounds > 1 ? rounds * (at_once * mean / ns * kTile + kBlock) : 0.0;
    const double join = ns > 1 ? 4.0 + double(T * H * D) * 8.0 * ns / 5e6 : 0.0;
    const double us = std::max(std::max(longest, sum), whole) + join;
    if (us < least * 0.95) least = us, best = ns;  // more splits where they gain something
  }
  return {best, int(tiles), nullptr, nullptr};
}
// The most splits of any bound up to kv_len: the model's choice goes up and down as the bound
// grows, but a buffer for the largest of several bounds has to be enough for all of them.
int most_splits(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t D, int64_t kv_len) {
  int most = 1;
  for (int64_t n = len_up(kv_len); n > 0 && split_limit(n) > most; n -= len_step(n - 1))
    most = std::max(most, plan(B, T, H, Hkv, D, n).nsplit);
  return most;
}
int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }
size_t ws_size(int nsplit, int64_t T, int64_t H, int64_t D) {
  return nsplit == 1 ? 0 : size_t(up256(nsplit * T * H * D * 4) + up256(nsplit * T * H * 8));
}

}  // namespace
}  // namespace ez

extern "C" size_t ezops_quant_prefill_attn_workspace_size(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t D,
                                                          int64_t kv_len) {
  if (B < 1 || T < 1 || T >= (int64_t(1) << 30) || H < 1 || H > 4096 || Hkv < 1 || H % Hkv || H / Hkv > 16 || D < 1 || D > 128 ||
      kv_len < 1)
    return 0;
  return ez::ws_size(ez::most_splits(B, T, H, Hkv, D, kv_len), T, H, D);
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
  const int rc = ez::check_attn8(op, a, page_size, block_size, H, Hkv, D, max_kv_len);
  if (rc != EZ_OK) return rc;
  ez::finish_args(a, page_size, max_kv_len);
  ez::SplitPlan pl = ez::plan(B, T, H, Hkv, D, a.cap);
  const int64_t blocks = int64_t(pl.tiles) * Hkv * pl.nsplit, joins = int64_t(pl.tiles) * Hkv * (ez::rows_of(D) * D / 1024);
  EZ_REQUIRE(blocks < int64_t(1) << 23 && (pl.nsplit == 1 || joins < int64_t(1) << 24), "%s: tokens * heads past one launch", op);
  if (pl.nsplit > 1) {
    const size_t need = ez::ws_size(pl.nsplit, T, H, D);
    EZ_REQUIRE(ws && ws_bytes >= need, "%s: workspace too small (%zu < %zu)", op, ws_bytes, need);
    EZ_REQUIRE(ez::kv8_aligned16(ws), "%s: workspace must be 16-byte aligned", op);
    for (const auto& x : ez::attn8_tensors(a, H))
      EZ_REQUIRE(!ez::overlap(ws, int64_t(need), x.p, x.n), "%s: workspace overlaps a tensor", op);
    pl.o = static_cast<float*>(ws);
    pl.ml = reinterpret_cast<float*>(static_cast<char*>(ws) + ez::up256(pl.nsplit * T * H * D * 4));
  }
#define EZ_GROUP(DD, TY, GG)                                                                                              \
  do {                                                                                                                    \
    hipLaunchKernelGGL((ez::quant_prefill_kernel<DD, TY, GG>), dim3(unsigned(blocks)), dim3(ez::waves_of(DD) * ez::kWave), 0, stream, \
                       a, pl);                                                                                            \
    if (pl.nsplit > 1)                                                                                                    \
      hipLaunchKernelGGL((ez::quant_prefill_join_kernel<DD, GG>), dim3(unsigned(joins)), dim3(256), 0, stream, a, pl);    \
  } while (0)
#define EZ_GO(DD, TY)                       \
  do {                                      \
    switch (H / Hkv) {                      \
      case 1: EZ_GROUP(DD, TY, 1); break;   \
      case 2: EZ_GROUP(DD, TY, 2); break;   \
      case 4: EZ_GROUP(DD, TY, 4); break;   \
      case 8: EZ_GROUP(DD, TY, 8); break;   \
      default: EZ_GROUP(DD, TY, 16); break; \
    }                                       \
  } while (0)
  EZ_KV8_DISPATCH(EZ_GO);
#undef EZ_GO
#undef EZ_GROUP
  return ez::launch_status(op);
}
