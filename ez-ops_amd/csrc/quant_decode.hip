// Attention of one token per sequence over the 8-bit KV cache.
//
//   s_j = scale * q . kc_j 2^(ek - 127),  o = sum_j softmax(s)_j vc_j 2^(ev - 127)
//
// kc, vc are the codes, ek, ev the exponents of the row's block (at least 16 rows each).
// The work is reading the codes once: 2 D bytes a row and kv head.
//
// A sequence is cut into chunks of rows; a block of 4 waves takes one chunk of one kv
// head for all G query heads of the group, so the codes cross memory once a group.
// Chunks are counted over the sequences' lengths on the device (block -> sequence, chunk
// by a wave scan), so a ragged batch is shared out by rows.  A wave's tiles of 32 rows
// lie 4 tiles apart.  Per tile:
//   * codes by 16-byte loads of whole rows, one tile ahead in registers, through the
//     wave's own LDS slab still in 8 bits
//   * S^T = K Q^T on v_mfma_f32_16x16x32_bf16: 16 rows of K (16 bytes of LDS a lane are two
//     operands, widened to bf16 in registers: int8 and e4m3 are exact there) against the
//     query heads, padded to 16 columns
//   * softmax in the exp2 domain, one head a lane column, scales as in the exponent:
//     w = 2^(c s' - m + v), c = scale log2(e) 2^(ek - 127), v = ev - 127: the weight times
//     the scale of v; l += w 2^-v
//   * O^T += V^T W^T, V^T by transposing 8-bit LDS reads (ds_read_b64_tr_b8) and widened
//     behind them; w as two bf16 parts, so that weights carry 16 significant bits
// The waves join (m, l, O) through LDS; a sequence of more than one chunk leaves fp32
// partials, which a second kernel joins.
//
// Measured: 32 sequences of 16384 rows, 32 / 8 heads of 128, e4m3: 162 us, 6.5 TB/s (a large
// copy reaches 5.1, a streaming read 6.7); 48 ragged ones of up to 4096 rows, 16 / 8 heads,
// int8: 41 us, 4.9 TB/s; one of 2000 rows 5.2 us and 3.5 to 5.5 for the join, both latency.
// Three waves a SIMD: four spill 13 registers (187 us for 173).
#include "common.h"
#include "internal.h"
#include "prof.h"
#include "quant_attn.h"
#include "status.h"
#include "../../include/ezops_hip.h"

namespace ez {

EZ_PROF_DEFINE(quantdecode)
namespace {

constexpr int kW = 4;              // waves of a block
constexpr int kT = 32;             // rows of a wave's tile
constexpr int kMaxSplits = 32;     // chunks of a sequence
constexpr int kSumSeqs = 1024;     // sequences whose lengths every block sums

struct SplitPlan {
  int target;       // chunks of a kv head to aim at; 0: a block per sequence
  int blocks;       // chunks at most
  float* o;         // partials [chunk][Hkv][G][D]
  float2* ml;       // [chunk][Hkv][G]
  int2* head;       // [B][Hkv]: block of a sequence's first chunk, number of chunks
};

__device__ __forceinline__ int seq_len(const QuantAttnArgs& a, int b) { return min(max(a.kv_lens[b], 0), int(a.cap)); }

// Rows of a chunk of a sequence of L rows, given the rows to aim at: equal ones, a whole
// number of tiles for every wave.
__device__ __forceinline__ int chunk_rows(int L, int aim) {
  const int n = min((L + aim - 1) / aim, kMaxSplits);
  return ((L + n - 1) / n + kW * kT - 1) / (kW * kT) * (kW * kT);
}
__device__ __forceinline__ int chunk_count(int L, int aim) {
  if (L <= aim) return 1;
  const int rows = chunk_rows(L, aim);
  return (L + rows - 1) / rows;
}

struct Chunk {
  int b, split, len, rows, count;
};

// The idx-th chunk of the batch; false behind the last one.  The rows to aim at are all the
// batch's over the chunks to aim at, so a ragged batch is shared out by rows.  A sequence
// without rows has one (which writes its zeros).
__device__ __forceinline__ bool find_chunk(const QuantAttnArgs& a, int target, int idx, Chunk& c) {
  constexpr int kPer = 4;  // lengths of a lane and step
  const int lane = threadIdx.x & (kWave - 1), B = int(a.B);
  if (B == 1) {  // the usual case of few blocks and little time
    c.len = seq_len(a, 0);
    const int aim = (c.len / target / (kW * kT) + 1) * (kW * kT);
    c.b = 0;
    c.split = idx;
    c.count = chunk_count(c.len, aim);
    c.rows = c.count == 1 ? c.len : chunk_rows(c.len, aim);
    return idx < c.count;
  }
  int L[kPer];
  auto lengths = [&](int b0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int s = b0 + kPer * lane + i;
      L[i] = s < B ? seq_len(a, s) : -1;
    }
  };
  float sum = 0.f;  // up to 2^10 lengths of 2^30
  for (int b0 = 0; b0 < B; b0 += kPer * kWave) {
    lengths(b0);
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += float(max(L[i], 0));
  }
  // Rounded up past the sum's rounding, so that the chunks stay within the blocks; from 2^30
  // on no sequence is longer.
  const float per = fminf(wave_reduce_uniform<false>(sum) * 1.0001f / float(target), 0x1p30f);
  const int aim = (int(per) / (kW * kT) + 1) * (kW * kT);
  for (int b0 = 0; b0 < B; b0 += kPer * kWave) {
    if (B > kPer * kWave) lengths(b0);
    int n[kPer], count = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      n[i] = L[i] < 0 ? 0 : chunk_count(L[i], aim);
      count += n[i];
    }
    const int end = wave_scan(count);
    const uint64_t hit = __ballot(idx < end);
    if (hit) {
      const int l = __ffsll(static_cast<unsigned long long>(hit)) - 1;
      int at = idx - (__builtin_amdgcn_readlane(end, l) - __builtin_amdgcn_readlane(count, l));
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int ni = __builtin_amdgcn_readlane(n[i], l);
        if (at >= 0 && at < ni) {
          c.b = b0 + kPer * l + i;
          c.split = at;
          c.len = __builtin_amdgcn_readlane(L[i], l);
          c.count = ni;
        }
        at -= ni;
      }
      c.rows = c.count == 1 ? c.len : chunk_rows(c.len, aim);
      return true;
    }
    idx -= __builtin_amdgcn_readlane(end, kWave - 1);
  }
  return false;
}

template <int D, int TYPE, int G>
__global__ __launch_bounds__(kW * kWave) __attribute__((amdgpu_waves_per_eu(3))) void quant_decode_kernel(QuantAttnArgs a,
                                                                                                         SplitPlan pl) {
  EZ_PROF_WAVE(kProfQuantAttnDecode);
  constexpr int CPR = D / 16;            // 16-byte chunks of a row of codes
  constexpr int RPL = kWave / CPR;       // rows of a load
  constexpr int NL = kT / RPL;           // loads of a tile
  constexpr int NX = D / 64;             // 16-byte operand pairs of a K row a lane
  constexpr int NDB = D / 16;            // 16-dim blocks of O^T
  struct Slabs {
    uint8_t K[kW][kT * D], V[kW][kT * D];  // [row][chunk ^ kswz(row)], [row][chunk ^ vswz(row)]
  };
  struct Joined {
    float O[kW][G][D], M[kW][G], L[kW][G];
  };
  __shared__ __align__(16) union {
    Slabs s;
    Joined j;
  } lds;
  // Chunk swizzles: 8 lanes that read one chunk of 8 rows (K), 16 lanes that read 16 bytes
  // of 8 rows (V), meet every bank once.
  auto kswz = [](int r) { return D == 128 ? r & 7 : (r >> 2) & 3; };
  auto vswz = [](int r) { return D == 128 ? ((r >> 1) & 1) | ((r >> 4) & 1) << 1 : (r >> 4) & 1; };

  const int kvh = int(blockIdx.x % unsigned(a.c.Hkv)), idx = int(blockIdx.x / unsigned(a.c.Hkv));
  Chunk ck{idx, 0, 0, 0, 1};
  if (pl.target == 0) ck.len = ck.rows = seq_len(a, idx);
  else if (!find_chunk(a, pl.target, idx, ck)) return;
  const int b = __builtin_amdgcn_readfirstlane(ck.b), split = __builtin_amdgcn_readfirstlane(ck.split);
  const int L = __builtin_amdgcn_readfirstlane(ck.len), rows = __builtin_amdgcn_readfirstlane(ck.rows);
  const int count = __builtin_amdgcn_readfirstlane(ck.count);
  if (pl.target != 0 && split == 0 && threadIdx.x == 0) pl.head[int64_t(b) * a.c.Hkv + kvh] = make_int2(int(blockIdx.x), count);
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, lg = lane >> 4;
  const int h0 = kvh * G;
  if (L == 0) {
    for (int i = threadIdx.x; i < G * D / 8; i += kW * kWave)
      *reinterpret_cast<uint4*>(a.out + (int64_t(b) * a.H + h0) * D + i * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  const int r0 = split * rows, r1 = min(L, r0 + rows), last = r1 - 1;

  // ---- loads of a tile: its page id one tile ahead (a vector load, so that it is waited
  // for in order with the codes), then codes and exponents
  const int32_t* table = a.table + int64_t(b) * a.M;
  const int pmask = (1 << a.c.page_sh) - 1;
  int lane0;
  asm volatile("v_mov_b32 %0, 0" : "=v"(lane0));
  auto start = [&](int t) { return t <= last ? t : last & ~(kT - 1); };  // tiles behind the end: the last one again
  auto page_id = [&](int t) { return table[(start(t) >> a.c.page_sh) + lane0]; };
  auto flat_row = [&](int t, int32_t id) {
    const uint32_t page = min(uint32_t(__builtin_amdgcn_readfirstlane(id)), uint32_t(a.c.num_pages - 1));
    return ((int64_t(page) * a.c.Hkv + kvh) << a.c.page_sh) + (start(t) & pmask);
  };
  uint4 kn[NL], vn[NL];
  int en;  // lanes 0, 1: exponents of the tile's two halves of K; 2, 3: of V
  auto load_k = [&](int t, int64_t at) {
    const int rows = last - start(t);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int p = i * RPL + lane / CPR;
      kn[i] = ld16_stream(a.c.K + (at + min(p, rows)) * D + ((lane % CPR) ^ kswz(p)) * 16);
    }
    en = ((lane & 2) ? a.c.Vs : a.c.Ks)[(at + 16 * (lane & 1)) >> a.c.block_sh];
  };
  auto load_v = [&](int t, int64_t at) {
    const int rows = last - start(t);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int p = i * RPL + lane / CPR;
      vn[i] = ld16_stream(a.c.V + (at + min(p, rows)) * D + ((lane % CPR) ^ vswz(p)) * 16);
    }
  };
  int t0 = r0 + wave * kT;
  int64_t at = flat_row(t0, page_id(t0));
  load_k(t0, at);
  load_v(t0, at);
  int32_t id = page_id(t0 + kW * kT);

  // Q operand of the pair (x, half): k-slot 8 lg + e is dim 64 x + 16 lg + 8 half + e, as K has it
  bf16x8_t qf[NX][2];
  {
    const uint16_t* qp = a.q + int64_t(b) * a.q_rs + int64_t(h0 + min(li, G - 1)) * D + 16 * lg;
#pragma unroll
    for (int x = 0; x < NX; ++x)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const uint4 v = *reinterpret_cast<const uint4*>(qp + 64 * x + 8 * f);
        qf[x][f] = as_bf16x8(li < G ? v : make_uint4(0, 0, 0, 0));
      }
  }
  uint8_t* ks = lds.s.K[wave];
  uint8_t* vs = lds.s.V[wave];
  int koff[NX], voff[NDB];
#pragma unroll
  for (int x = 0; x < NX; ++x) koff[x] = li * D + (((4 * x + lg) ^ kswz(li)) * 16);
  static_assert(kT == 32, "the swizzle of K row 16 + li is that of li");
  {
    const int i = li >> 1, row = 4 * lg + (i & 3) + 16 * (i >> 2);
#pragma unroll
    for (int d = 0; d < NDB; ++d) voff[d] = row * D + ((d ^ vswz(row)) * 16) + 8 * (li & 1);
  }

  // Lane (li, lg): head li's reference m, its share of the sum, O^T[16 d + 4 lg + r][li] in o[d][r]
  float m = kLowest, l = 0.f;
  f32x4_t o[NDB];
#pragma unroll
  for (int d = 0; d < NDB; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  for (; t0 < r1; t0 += kW * kT) {
    const int tn = t0 + kW * kT;
    const bool tail = t0 + kT > r1;
#pragma unroll
    for (int i = 0; i < NL; ++i) *reinterpret_cast<uint4*>(ks + (i * kWave + lane) * 16) = kn[i];
    const int e = kv8_exp(en);
    const float cv = lane & 2 ? (e == kKvNanExp ? __uint_as_float(0x7fc00000u) : float(e - 127)) : kv8_factor(a.scale, e);
    const int iv = e == kKvNanExp ? 127 : 254 - e;
    at = flat_row(tn, id);
    load_k(tn, at);
    id = page_id(tn + kW * kT);
    f32x4_t s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < NX; ++x) {
        const uint4 k = *reinterpret_cast<const uint4*>(ks + 16 * u * D + koff[x]);
        const uint2 w0 = kv8_bf16x4<TYPE>(k.x), w1 = kv8_bf16x4<TYPE>(k.y), w2 = kv8_bf16x4<TYPE>(k.z), w3 = kv8_bf16x4<TYPE>(k.w);
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(make_uint4(w0.x, w0.y, w1.x, w1.y)), qf[x][0], s[u], 0, 0, 0);
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(make_uint4(w2.x, w2.y, w3.x, w3.y)), qf[x][1], s[u], 0, 0, 0);
      }
    }
    // s[u][r] = s' of (head li, row t0 + 16 u + 4 lg + r)
    float c[2], v[2], inv[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      c[u] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(cv), u));
      v[u] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(cv), 2 + u));
      inv[u] = __int_as_float(__builtin_amdgcn_readlane(iv, 2 + u) << 23);
    }
    if (tail) {
      if (t0 + 16 >= r1) c[1] = 1.f, v[1] = 0.f;  // no row of this half: its exponents may be anything
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (t0 + 16 * u + 4 * lg + r >= r1) s[u][r] = -INFINITY;
    }
    float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])) * c[0],
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])) * c[1]);
    mx = colgroup_max(mx);
    if (__builtin_amdgcn_ballot_w64(mx > m)) {  // rescale only where a reference moves
      const float mn = fmaxf(m, mx);
      const float alpha = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < NDB; ++d) o[d] *= alpha;
    }
    // W^T operand: k-slot 8 lg + e is row 16 (e / 4) + 4 lg + e % 4, w = hi + lo in bf16
    uint32_t wh[4], wl[4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float off = v[u] - m;
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[u][2 * q], c[u], off));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[u][2 * q + 1], c[u], off));
        wh[2 * u + q] = cvt_bf2(p0, p1);
        wl[2 * u + q] = cvt_bf2(p0 - bf_lo(wh[2 * u + q]), p1 - bf_hi(wh[2 * u + q]));
        sum += p0 + p1;
      }
      l = fmaf(sum, inv[u], l);
    }
    const bf16x8_t ph = as_bf16x8(make_uint4(wh[0], wh[1], wh[2], wh[3]));
    const bf16x8_t pw = as_bf16x8(make_uint4(wl[0], wl[1], wl[2], wl[3]));

    if (tail) {  // rows behind the end weigh 0, but 0 * NaN would not: they are zeros
#pragma unroll
      for (int i = 0; i < NL; ++i)
        if (t0 + i * RPL + lane / CPR >= r1) vn[i] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) *reinterpret_cast<uint4*>(vs + (i * kWave + lane) * 16) = vn[i];
    load_v(tn, at);
#pragma unroll
    for (int d = 0; d < NDB; ++d) {
      typedef int i32x2_t __attribute__((ext_vector_type(2)));
      const i32x2_t x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2_t*)(vs + voff[d]));
      const uint2 w0 = kv8_bf16x4<TYPE>(uint32_t(x[0])), w1 = kv8_bf16x4<TYPE>(uint32_t(x[1]));
      const bf16x8_t va = as_bf16x8(make_uint4(w0.x, w0.y, w1.x, w1.y));
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, ph, o[d], 0, 0, 0);
      o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pw, o[d], 0, 0, 0);
    }
  }

  // ---- join the waves: each writes (m, l, O), then a thread takes 4 dims of a head
  l = rowgroup_sum<16>(l);
  __syncthreads();  // the slabs are read no more
  if (li < G) {
#pragma unroll
    for (int d = 0; d < NDB; ++d)
      *reinterpret_cast<float4*>(&lds.j.O[wave][li][16 * d + 4 * lg]) = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
    if (lg == 0) {
      lds.j.M[wave][li] = m;
      lds.j.L[wave][li] = l;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < G * D / 4; i += kW * kWave) {
    const int h = i / (D / 4), d = i % (D / 4) * 4;
    float M = kLowest;
#pragma unroll
    for (int w = 0; w < kW; ++w) M = fmaxf(M, lds.j.M[w][h]);
    float ov[4] = {0.f, 0.f, 0.f, 0.f}, lv = 0.f;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      const float f = __builtin_amdgcn_exp2f(lds.j.M[w][h] - M);
      lv = fmaf(f, lds.j.L[w][h], lv);
#pragma unroll
      for (int k = 0; k < 4; ++k) ov[k] = fmaf(f, lds.j.O[w][h][d + k], ov[k]);
    }
    const int64_t hq = int64_t(b) * a.H + h0 + h;
    if (count == 1) {
      const float r = 1.f / lv;
      *reinterpret_cast<uint2*>(a.out + hq * D + d) = make_uint2(cvt_bf2(ov[0] * r, ov[1] * r), cvt_bf2(ov[2] * r, ov[3] * r));
    } else {
      const int64_t part = int64_t(blockIdx.x) * G + h;
      *reinterpret_cast<float4*>(pl.o + part * D + d) = make_float4(ov[0], ov[1], ov[2], ov[3]);
      if (d == 0) pl.ml[part] = make_float2(M, lv);
    }
  }
}

// Joins the chunks of a (sequence, query head): 4 dims a thread.  Sequences of one chunk
// are written already.
template <int D>
__global__ __launch_bounds__(256) void quant_decode_join_kernel(QuantAttnArgs a, SplitPlan pl) {
  EZ_PROF_WAVE(kProfQuantAttnCombine);
  constexpr int TPR = D / 4;
  const int64_t hq = int64_t(blockIdx.x) * (256 / TPR) + threadIdx.x / TPR;
  if (hq >= a.B * a.H) return;
  const int d = int(threadIdx.x) % TPR * 4, G = a.H / a.c.Hkv;
  const int2 head = pl.head[hq / G];
  if (head.y == 1) return;
  const int64_t part = int64_t(head.x) * G + hq % G, step = int64_t(a.c.Hkv) * G;
  const float4* po = reinterpret_cast<const float4*>(pl.o + part * D + d);
  float o[4];
  if (head.y <= 4) join_parts<4>(pl.ml + part, po, step, step * (D / 4), head.y, o);
  else join_parts<16>(pl.ml + part, po, step, step * (D / 4), head.y, o);
  *reinterpret_cast<uint2*>(a.out + hq * D + d) = make_uint2(cvt_bf2(o[0], o[1]), cvt_bf2(o[2], o[3]));
}

// Chunks of a kv head to aim at: what fills the three places that a CU has for blocks, less
// the half chunk that a sequence adds on average (two places where a sequence would get more
// chunks than the join takes at once: 4 x 8192 rows of 32 / 8 heads 38.7 to 35.8 us); with many sequences,
// chunks of twice the mean length, so that a long one among them is shared out.  None below a
// tile a wave.  Sequences that are short and fill the card whole stay whole, without a join
// (64 x 1024 rows 42.7 to 38 us, 200 of up to 1500 79 to 71), and so do more than 1024.
SplitPlan plan(int64_t B, int64_t Hkv, int64_t kv_len) {
  const int64_t cus = num_cus();
  if (kv_len <= kW * kT || B > kSumSeqs || (B * Hkv >= 2 * cus && kv_len <= 2048)) return {0, int(B), nullptr, nullptr, nullptr};
  int64_t places = 3 * cus / Hkv;
  if (places > 16 * B) places = 2 * cus / Hkv > 16 * B ? 2 * cus / Hkv : 16 * B;
  int64_t target = places - B / 2 > B / 2 ? places - B / 2 : B / 2;
  target = target < 1 ? 1 : target;
  int64_t most = (kv_len + kW * kT - 1) / (kW * kT);  // of a sequence
  most = most < kMaxSplits ? most : kMaxSplits;
  const int64_t blocks = target + B < B * most ? target + B : B * most;
  return {int(target), int(blocks), nullptr, nullptr, nullptr};
}
int64_t up256(int64_t x) { return (x + 255) / 256 * 256; }
size_t ws_size(const SplitPlan& pl, int64_t B, int64_t H, int64_t Hkv, int64_t D) {
  return pl.target == 0 ? 0 : size_t(up256(pl.blocks * H * D * 4) + up256(pl.blocks * H * 8) + up256(B * Hkv * 8));
}

}  // namespace
}  // namespace ez

extern "C" size_t ezops_quant_paged_attn_decode_workspace_size(int64_t B, int64_t H, int64_t Hkv, int64_t D,
                                                               int64_t kv_len) {
  if (B < 1 || B > 65536 || H < 1 || H > 4096 || Hkv < 1 || H % Hkv || D < 1 || D > 128 || kv_len < 1) return 0;
  const int64_t most = int64_t(1) << 30;  // rows of a table; the size grows with the bound up to there
  return ez::ws_size(ez::plan(B, Hkv, kv_len < most ? kv_len : most), B, H, Hkv, D);
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
  const int rc = ez::check_attn8(op, a, page_size, block_size, H, Hkv, D, max_kv_len);
  if (rc != EZ_OK) return rc;
  ez::finish_args(a, page_size, max_kv_len);
  ez::SplitPlan pl = ez::plan(B, Hkv, a.cap);
  const int64_t blocks = Hkv * pl.blocks, joins = (B * H * (D / 4) + 255) / 256;
  EZ_REQUIRE(blocks < int64_t(1) << 24, "%s: batch * heads past one launch", op);
  if (pl.target) {
    const size_t need = ez::ws_size(pl, B, H, Hkv, D);
    EZ_REQUIRE(ws && ws_bytes >= need, "%s: workspace too small (%zu < %zu)", op, ws_bytes, need);
    EZ_REQUIRE(ez::kv8_aligned16(ws), "%s: workspace must be 16-byte aligned", op);
    for (const auto& x : ez::attn8_tensors(a, H))
      EZ_REQUIRE(!ez::overlap(ws, int64_t(need), x.p, x.n), "%s: workspace overlaps a tensor", op);
    char* at = static_cast<char*>(ws);
    pl.o = reinterpret_cast<float*>(at);
    pl.ml = reinterpret_cast<float2*>(at += ez::up256(pl.blocks * H * D * 4));
    pl.head = reinterpret_cast<int2*>(at += ez::up256(pl.blocks * H * 8));
  }
#define EZ_GROUP(DD, TY, GG)                                                                                                  \
  hipLaunchKernelGGL((ez::quant_decode_kernel<DD, TY, GG>), dim3(unsigned(blocks)), dim3(ez::kW * ez::kWave), 0, stream, a, pl)
#define EZ_GO(DD, TY)                                                                                                         \
  do {                                                                                                                        \
    switch (H / Hkv) {                                                                                                        \
      case 1: EZ_GROUP(DD, TY, 1); break;                                                                                     \
      case 2: EZ_GROUP(DD, TY, 2); break;                                                                                     \
      case 4: EZ_GROUP(DD, TY, 4); break;                                                                                     \
      case 8: EZ_GROUP(DD, TY, 8); break;                                                                                     \
      default: EZ_GROUP(DD, TY, 16); break;                                                                                   \
    }                                                                                                                         \
    if (pl.target)                                                                                                            \
      hipLaunchKernelGGL((ez::quant_decode_join_kernel<DD>), dim3(unsigned(joins)), dim3(256), 0, stream, a, pl);             \
  } while (0)
  EZ_KV8_DISPATCH(EZ_GO);
#undef EZ_GO
#undef EZ_GROUP
  return ez::launch_status(op);
}
