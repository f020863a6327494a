// Attention over the quantized cache for few query rows (single tokens, drafts): streams the cache once.
//
// Mathematics. For a KV head's query rows r (its query heads times the query tokens) and keys j,
//   x_rj = scale * sum_b dk_jb * (sum_{i in b} Q_ri (k_ji - off)),   o_r = sum_j 2^(x_rj log2e - ref) dv_jb (v_ji - off) / L
// in one pass, with a running reference exponent `ref` and sum L for each row. The quants are whole numbers, so both
// products run on the tensor cores (16x8x16, f16 in, f32 sums) with keys and values as the 16-row operand and 8 query
// rows as the columns: nothing is padded, and no quant is rounded. What an operand's 16 bits hold:
//   - keys (16-bit calls): the quant's bits alone, i.e. the f16 subnormal q * 2^-24 (or q * 2^-20 for a nibble left in bits 4-7): one
//     AND unpacks two values. The offset -off * sum(Q) of a block is a constant of the row, added to the block's sum.
//   - queries: scaled by a power of two to 2^13..2^14; f32 queries take two parts. 16-bit queries are exact where a row's
//     values lie within 2^27 (f16; bf16 2^30; q4_0 keys' high nibbles take a 16th: 2^23 and 2^26), smaller ones are within
//     2^-38 (2^-34) of its largest.
//     A block's scale dk (per key and block) multiplies the f32 sum of the block.
//   - values: the quant minus its offset, again as an exact subnormal (an addition more for two values): offsets taken
//     off the sums instead would cancel there, and leave their cut-off bits.
//   - weights: 2^(x - ref) * dv in f32 for each block, rounded once to f16 (f32 calls: two parts, 22 bits). `ref` follows
//     the row's scores and the value scales, so that the products stay at most 2^15 and a row's largest near 2^8: they
//     cannot overflow whatever the scales, and lose no bits to f16's small exponents until 2^-22 of the largest.
// A weight matrix leaves the first product with keys along the lanes' rows and enters the second with keys along their
// pairs: one 8x8 transpose in registers each.
//
// What bounds it: latency, with the cache's bytes and the unpacking close behind each other: no unit is above 60% (issue
// 59%, ALU 48%, DRAM 50%) at the 12 warps an SM that 168 registers leave. The CTAs fill the GPU once and take equal shares of
// all stages (16 to 64 keys) of all sequences, heads and row tiles, whatever their lengths; a tile's stages go round the four
// warps, each with a ring of its own, and the warps join at the tile's end. Tiles that cross shares are joined by a second
// kernel. Measured: 8 sequences of 90001 to 131072 keys, 64 query heads on 8 of 128, f16: 231 us in a long run with three such
// caches in turn (4.4 TB/s), 200 at best; 64 sequences of 100 to 8192 keys: 80 us (3.8 TB/s), of which about 15 us are
// beginnings and ends. Without its arithmetic the first takes 158 us, without its copies 193 us. What did not help: 16 warps
// of 128 registers (a stage of 32 keys then: 262 us), every warp on its own (225 us; its instructions come from farther
// away), bulk copies instead of cp.async (the same), the next keys' scores beside these keys' products (229 us).
#pragma once

#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

#include "kv_device.cuh"
#include "kv_internal.h"
#include "tc_device.cuh"

namespace b2q {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNoRef = -1e30f;  // reference exponent of a row that has seen no key

template <int FMT, int NB>
struct KvTile {
  static constexpr int kRow = NB * (FMT == 0 ? 16 : 32);  // quant bytes of a token's row
  // tokens a stage: at most 9216 bytes, so that 12 warps with two stages (four of the
  // smallest rows) each fill an SM
  static constexpr int kTokens = kRow <= 64 ? 64 : (kRow <= 128 ? 32 : 16);
  static constexpr int kQuants = kTokens * kRow, kScales = kTokens * NB * 2;
  static constexpr int kStage = 2 * (kQuants + kScales);
  static constexpr int kWarps = 4;
  static constexpr int kStages = kRow <= 32 ? 4 : 2;
  static constexpr int kRing = kStage * kStages * kWarps;
};

// CTAs an SM: as many as their registers and rings leave room for.
template <int FMT, int NB, int NT, int PARTS>
constexpr int kv_ctas_per_sm() {
  return NB == 8 || NT == 2 || (PARTS == 2 && NB > 2) ? 2 : 3;
}

// Row r of a 16-token tile is this token: chosen so that both the key loads (lanes of two rows side by side) and the
// value loads (lanes of four tokens side by side) spread over the shared-memory banks.
__device__ __forceinline__ int tile_token(int r) { return (r & 1) ? ((r >> 1) ^ 1) + 4 : (r >> 1); }

// N consecutive 32-bit words of shared memory.
template <int N>
__device__ __forceinline__ void lds_words(const uint8_t* at, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(at + 4 * i);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(at + 4 * i);
      w[i] = v.x, w[i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = *reinterpret_cast<const uint32_t*>(at + 4 * i);
  }
}

// N consecutive 16-bit words, two to a register (the last register's high half is unused when N is odd).
template <int N>
__device__ __forceinline__ void lds_halves(const uint8_t* at, uint32_t (&w)[(N + 1) / 2]) {
  if constexpr (N % 2 == 0) {
    lds_words<N / 2>(at, w);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t h = *reinterpret_cast<const uint16_t*>(at + 2 * i);
      w[i / 2] = (i & 1) ? (w[i / 2] | h << 16) : h;
    }
  }
}

// The NB f16 scales of a token.
template <int NB>
__device__ __forceinline__ void lds_scales(const uint8_t* at, float (&d)[NB]) {
  uint32_t w[(NB + 1) / 2];
  lds_halves<NB>(at, w);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const __half2 h = *reinterpret_cast<const __half2*>(&w[b / 2]);
    d[b] = (b & 1) ? __high2float(h) : __low2float(h);
  }
}

// Quants as pairs of f16, from 16 bits each of a register: the nibbles of bits 0-3 or of bits 4-7 (worth 16 each), or the
// bytes 0, 1 or 2, 3 of a word. SIGNED: the quant less its offset, as a normal number. Else the quant's bits alone, the
// subnormal of 2^-24 times it, in one instruction; but the tensor cores take the exponent of a subnormal as 2^-14 where
// they align a sum's terms, which costs up to 10 of the sum's bits (measured, f32 calls: error 5e-6, and 5e-7 so).
template <bool SIGNED>
__device__ __forceinline__ uint32_t low_nibbles(uint32_t w) {
  return SIGNED ? add_half2((w & 0x000f000fu) | 0x64006400u, 0xe408e408u) : w & 0x000f000fu;  // 1024 + q - 1032
}
template <bool SIGNED>
__device__ __forceinline__ uint32_t high_nibbles(uint32_t w) {
  return SIGNED ? add_half2((w & 0x00f000f0u) | 0x64006400u, 0xe480e480u) : w & 0x00f000f0u;  // 1024 + 16 q - 1152
}
template <bool SIGNED>
__device__ __forceinline__ uint32_t two_bytes(uint32_t w, int upper) {
  return SIGNED ? add_half2(__byte_perm(w, 0x64646464u, upper ? 0x4342 : 0x4140), 0xe480e480u)  // 1024 + u - 1152
                : __byte_perm(w, 0, upper ? 0x4342 : 0x4140);
}

// 4 values at p (of type dtype, p counted in elements), 4-element aligned.
__device__ __forceinline__ void load4_as(const void* p, int64_t i, int dtype, float (&v)[4]) {
  if (dtype == B2Q_DTYPE_F32)
    load4(static_cast<const float*>(p) + i, v);
  else if (dtype == B2Q_DTYPE_F16)
    load4(static_cast<const __half*>(p) + i, v);
  else
    load4(static_cast<const __nv_bfloat16*>(p) + i, v);
}
__device__ __forceinline__ void store4_as(void* p, int64_t i, int dtype, float a, float b, float c, float d) {
  if (dtype == B2Q_DTYPE_F32)
    store4(static_cast<float*>(p) + i, a, b, c, d);
  else if (dtype == B2Q_DTYPE_F16)
    store4(static_cast<__half*>(p) + i, a, b, c, d);
  else
    store4(static_cast<__nv_bfloat16*>(p) + i, a, b, c, d);
}

__device__ __forceinline__ void store_elt(void* p, int64_t i, int dtype, float v) {
  if (dtype == B2Q_DTYPE_F32)
    static_cast<float*>(p)[i] = v;
  else if (dtype == B2Q_DTYPE_F16)
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// tanh(z) / z of u = z^2 for |z| <= 0.6: fitted to the smallest largest relative error (9.0e-8 with the constants as they
// stand in f32, 1.8e-7 with the steps' roundings). Beyond, tanh(|z|) = 1 - 2 / (e^2z + 1); scores near the cap are rare, and where a warp has none it skips that (two of the slow units' steps).
constexpr float kTanhLimit = 0.6f;
constexpr float kTanh0 = 0.99999994f, kTanh1 = -0.3333231f, kTanh2 = 0.13310172f, kTanh3 = -0.05210143f, kTanh4 = 0.015475366f;
__device__ __forceinline__ float tanh_near(float z) {
  const float u = z * z;
  return z * fmaf(u, fmaf(u, fmaf(u, fmaf(u, kTanh4, kTanh3), kTanh2), kTanh1), kTanh0);
}
__device__ __forceinline__ float tanh_far(float z) {
  return copysignf(1.f - __fdividef(2.f, exp2_approx(fabsf(z) * (2.f * kLog2e)) + 1.f), z);
}

// Sequence b's query tokens (held within q whatever cu_q says), its length, which the queries' positions go by, and what of
// it the table holds, past which no key is visible.
struct Sequence {
  int64_t q0;
  int n, end, len;
};
__device__ __forceinline__ Sequence sequence(const AttnParams& p, int b) {
  Sequence s = {b, 1, 0, 0};
  if (p.cu_q) {
    s.q0 = max((int64_t)0, min((int64_t)p.cu_q[b], p.T));
    s.n = (int)(min((int64_t)p.cu_q[b + 1], p.T) - s.q0);
  }
  s.end = max(0, p.lens[b]);
  s.len = min(s.end, p.table_pages << p.page_shift);
  return s;
}

// Position and visible keys [lo, hi) of query i of sequence b.
struct QuerySpan {
  int pos, lo, hi;
};
__device__ __forceinline__ QuerySpan query_span(const AttnParams& p, int b, int i, const Sequence& q) {
  QuerySpan s;
  s.pos = q.end - q.n + i;
  s.hi = s.pos + 1;
  if (p.prefix) s.hi = max(s.hi, p.prefix[b]);
  s.hi = max(0, min(s.hi, q.len));
  s.lo = p.starts ? max(0, p.starts[q.q0 + i]) : 0;
  if (p.window > 0 && s.pos >= p.window) s.lo = max(s.lo, s.pos - p.window + 1);
  return s;
}

// What beginning a tile costs a CTA, in stages of its share: without it, a share of many short tiles takes far longer than
// one long run. Measured with costs of 4 / 8 / 12 / 24, us, bf16, 32 heads on 8: 64 sequences of 100 to 8192 tokens, q4_0
// heads of 128 88 / 80 / 81 / 86, of 256 173 / 160 / 154 / 158, four tokens each of 48 such 131 / 117 / 99 / 105, 300 of 20
// to 2048 133 / 123 / 118 / 126 and in q8_0 154 / 138 / 131 / 139; f32 (whose
// stages take longer), heads of 128 128 / 122 / 124 / 131, five tokens each of 16 of 7 to 6001, heads of 64: 37 with 8, 40
// with 12.
template <int PARTS>
constexpr int kTileCost = PARTS == 2 ? 8 : 12;

// The stages that hold the visible keys of row tile rt of sequence b: `count` is 0 for a tile without rows and at least 1
// for any other, so that a tile that sees nothing is somebody's work too.
struct Span {
  int first, count;
};
// One thread's answer, or (WARP) a warp's for the same tile, its lanes sharing the queries.
template <int STG, int R, bool WARP = false>
__device__ __forceinline__ Span tile_span(const AttnParams& p, int b, int rt) {
  const Sequence q = sequence(p, b);
  if (rt * R >= q.n * p.group) return {0, 0};
  int i0 = 0, i1 = 0;
  if (p.cu_q) i0 = rt * R / p.group, i1 = min(q.n - 1, (rt * R + R - 1) / p.group);
  int lo = INT_MAX, hi = 0;
  if (!p.starts) {  // both ends grow with the position
    lo = query_span(p, b, i0, q).lo, hi = query_span(p, b, i1, q).hi;
  } else {
#pragma unroll 4
    for (int i = i0 + (WARP ? (int)(threadIdx.x & 31) : 0); i <= i1; i += WARP ? 32 : 1) {
      const QuerySpan s = query_span(p, b, i, q);
      if (s.lo < s.hi) lo = min(lo, s.lo), hi = max(hi, s.hi);
    }
    if (WARP) lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi);
  }
  if (lo >= hi) return {0, 1};
  return {lo / STG, (hi + STG - 1) / STG - lo / STG};
}

// A tile's units of a share: `cost` without stages, then its stages.
__device__ __forceinline__ int tile_units(Span s, int cost) { return s.count ? s.count + cost : 0; }

// The plan: every CTA an equal share of all stages. Entries (sequence, row tile) have their stages, after cost units without
// any, once a KV head; a CTA's share is [pos, end) of their run, at least `least` units (unless none are left),
// and begins `skip` units into the tile of (entry, head). All W warps call it; the scratch is read until the barrier
// that ends it.
struct Share {
  int64_t per, pos, end;
  int entry, head, skip;
};
template <int W>
struct ShareScratch {
  int64_t scan[W];
  int entry, head, skip;
};
template <int STG, int R, int W>
__device__ __forceinline__ Share plan_share(const AttnParams& p, int cost, int least, ShareScratch<W>& scratch) {
  constexpr int kThreads = W * 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int entries = p.batch * p.row_tiles, chunk = (entries + kThreads - 1) / kThreads;
  const int e0 = min(entries, (int)threadIdx.x * chunk), e1 = min(entries, e0 + chunk);
  Share s;
  int64_t mine = 0;
  for (int e = e0; e < e1; ++e) mine += tile_units(tile_span<STG, R>(p, e / p.row_tiles, e % p.row_tiles), cost);
  mine *= p.heads;
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) scratch.scan[warp] = upto;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < warp) upto += scratch.scan[w];
    total += scratch.scan[w];
  }
  if (total < (int64_t)1 << 31)
    s.per = max((int)((uint32_t)(total + gridDim.x - 1) / gridDim.x), least);
  else
    s.per = (total + gridDim.x - 1) / gridDim.x;
  s.pos = s.per * blockIdx.x;
  s.end = min(total, s.pos + s.per);
  if (s.pos < s.end && s.pos >= upto - mine && s.pos < upto) {  // the thread whose entries hold the beginning
    int64_t off = s.pos - (upto - mine);
    for (int e = e0; e < e1; ++e) {
      const int count = tile_units(tile_span<STG, R>(p, e / p.row_tiles, e % p.row_tiles), cost);
      if (off < (int64_t)count * p.heads) {
        int h = 0;
        while (off >= count) off -= count, ++h;
        scratch.entry = e, scratch.head = h, scratch.skip = (int)off;
        break;
      }
      off -= (int64_t)count * p.heads;
    }
  }
  __syncthreads();
  s.entry = scratch.entry, s.head = scratch.head, s.skip = scratch.skip;
  return s;
}

// FMT 0 (q4_0) or 2 (q8_0), NB blocks a head, NT tiles of 8 query rows, PARTS f16 parts of queries and weights.
template <int FMT, int NB, int NT, int PARTS>
__global__ void __launch_bounds__(128, (kv_ctas_per_sm<FMT, NB, NT, PARTS>())) attention_kernel(const AttnParams p) {
  using C = KvTile<FMT, NB>;
  constexpr int D = NB * 32, W = C::kWarps, S = C::kStages, STG = C::kTokens, SUB = STG / 16, R = NT * 8;
  constexpr int kCost = kTileCost<PARTS>;
  constexpr bool SIGNED = PARTS == 2;  // quants enter the products with their offset taken off
  constexpr float kOff = FMT == 0 ? 8.f : 128.f;
  constexpr int UN = SUB % 2 == 0 && NB * NT <= 4 && PARTS == 1 ? 2 : 1;
  extern __shared__ __align__(128) uint8_t smem[];  // [stage][warp] ring; the last stage holds the queries at first
  __shared__ int s_lo[R], s_hi[R], s_pos[R], s_out[R], s_top[R];
  __shared__ float s_slope[R], s_rowf[R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  uint8_t* const ring = smem + warp * C::kStage;  // stage s of this warp: s * W stages on
  pdl_wait_then_trigger();

  __shared__ ShareScratch<W> plan;
  const Share share = plan_share<STG, R, W>(p, kCost, W, plan);
  const int64_t per = share.per, end = share.end;
  int64_t pos = share.pos;
  if (pos >= end) {
    if (threadIdx.x == 0) p.joins[blockIdx.x].first = -1;
    return;
  }
  int entry = share.entry, h = share.head, skip = share.skip;
  AttnJoin join = {-1, 0, 0, 0, 0};

  const int page = 1 << p.page_shift, piece_shift = min(p.page_shift, __ffs(STG) - 1);
  const int pieces = STG >> piece_shift;  // a stage's contiguous pieces, each of a page
  const bool special = p.softcap > 0.f || p.slopes != nullptr;
  const int tokA = tile_token(g);  // key rows g and g + 8 of a tile: tokA, tokA + 8
  const int vtok0 = tile_token(2 * t), vtok1 = tile_token(2 * t + 1);

  while (pos < end) {
    // -------------------------------------------------------------- the next tile of the share: (b, rt, h), its rows
    const int b = p.row_tiles == 1 ? entry : entry / p.row_tiles, rt = entry - b * p.row_tiles;
    const Span span = tile_span<STG, R, true>(p, b, rt);
    if (h == p.heads || span.count == 0) {
      ++entry, h = 0;
      continue;
    }
    const int units = tile_units(span, kCost), take = (int)min((int64_t)(units - skip), end - pos);
    // this share's stages of the tile: [from, to) of span.count
    const int from = max(0, skip - kCost), to = max(0, skip + take - kCost);
    if (to == from) {
      pos += take, skip += take;
      if (skip == units) skip = 0, ++h;
      continue;
    }
    const Sequence q = sequence(p, b);
    const int rows = q.n * p.group - rt * R;  // rows from this tile on (at least 1)
    if (threadIdx.x == 0 && (q.end > q.len || (rt + 1 == p.row_tiles && rows > R)))
      atomicCAS(&g_device_error, 0, q.end > q.len ? kErrPage : kErrQueries);
    const int begin = span.first + from, stop = span.first + to;

    const int32_t* table = p.table + (int64_t)b * p.table_stride;
    // the page of piece `lane` of a stage, or -1
    auto page_of = [&](int stage) -> int {
      const int tok = stage * STG + (lane << piece_shift);
      if (stage >= stop || lane >= pieces || tok >= q.len) return -1;
      const int id = table[tok >> p.page_shift];
      if (id < 0 || id >= p.pages) {
        atomicCAS(&g_device_error, 0, kErrPage);
        return -1;
      }
      return id;
    };
    // copies a stage into ring slot s, 16 bytes a lane at a time; pieces without a page are filled with zeros
    auto copy = [&](int stage, int s, int id) {
      const uint32_t to = smem_addr(ring + s * (W * C::kStage)) + lane * 16;
      if (stage < stop) {
        if (pieces == 1) {
          const int one = __shfl_sync(0xffffffffu, id, 0);
          const bool is = one >= 0;
          const int64_t row = is ? (((int64_t)one * p.heads + h) << p.page_shift) + ((stage * STG) & (page - 1)) : 0;
          const uint8_t* k = p.kq + row * C::kRow + lane * 16;
          const uint8_t* v = p.vq + row * C::kRow + lane * 16;
#pragma unroll
          for (int j = 0; j < C::kQuants; j += 512) cp_async16(to + j, k + j, is);
#pragma unroll
          for (int j = 0; j < C::kQuants; j += 512) cp_async16(to + C::kQuants + j, v + j, is);
          if (lane * 16 < C::kScales) {
            cp_async16(to + 2 * C::kQuants, reinterpret_cast<const uint8_t*>(p.ks + row * NB) + lane * 16, is);
            cp_async16(to + 2 * C::kQuants + C::kScales, reinterpret_cast<const uint8_t*>(p.vs + row * NB) + lane * 16,
                       is);
          }
        } else {
          // chunk c of a plane: its token, that token's piece and page
          auto chunk = [&](int c, int row_bytes, const uint8_t* a, const uint8_t* b, uint32_t to_a, uint32_t to_b) {
            const int tok = c * 16 / row_bytes, pc = tok >> piece_shift;
            const int one = __shfl_sync(0xffffffffu, id, pc & 31);
            const bool is = one >= 0 && pc < pieces;
            const int64_t row = is ? ((int64_t)one * p.heads + h) << p.page_shift : 0;
            const int64_t src = row * row_bytes + (is ? c * 16 - (pc << piece_shift) * row_bytes : 0);
            if (pc < pieces) cp_async16(to_a, a + src, is), cp_async16(to_b, b + src, is);
          };
#pragma unroll 1
          for (int j = 0; j < C::kQuants; j += 512)
            chunk(j / 16 + lane, C::kRow, p.kq, p.vq, to + j, to + C::kQuants + j);
          chunk(lane, NB * 2, reinterpret_cast<const uint8_t*>(p.ks), reinterpret_cast<const uint8_t*>(p.vs),
                to + 2 * C::kQuants, to + 2 * C::kQuants + C::kScales);
        }
      }
      cp_async_commit();  // a group a stage, empty past the last
    };
    // a page that cannot be read masks its tokens: bit i of a stage's word is whether piece i was
    const uint32_t full = (1u << pieces) - 1;
    uint32_t good[S];
    int ids[S];
#pragma unroll
    for (int i = 0; i < S; ++i) ids[i] = page_of(begin + warp + i * W);
#pragma unroll
    for (int i = 0; i < S; ++i) {
      good[i] = __ballot_sync(0xffffffffu, ids[i] >= 0);
      if (i + 1 < S) copy(begin + warp + i * W, i, ids[i]);
    }

    // -------------------------------------------------------------- queries: the tile's rows as B operands of f16
    // A thread takes 8 values of a row at a time. Rows are scaled by a power of two; block sums give the start values.
    // Operands lie in the ring's last stage as [part][row][block][t] 16-byte words, one for a lane's 4 registers.
    uint4* sq = reinterpret_cast<uint4*>(smem + (S - 1) * W * C::kStage);
    float* s_start = reinterpret_cast<float*>(sq + PARTS * R * NB * 4);  // [row][block]
    static_assert(PARTS * R * NB * 4 * 16 + R * NB * 4 <= W * C::kStage, "queries in one stage of the ring");
    constexpr int kItems = R * NB * 4, kPasses = (kItems + 127) / 128;
    if (threadIdx.x < R) {
      const int r = threadIdx.x, rr = rt * R + (r < rows ? r : 0);
      const int i = p.cu_q ? rr / p.group : 0, head = h * p.group + (rr - i * p.group);
      const QuerySpan s = query_span(p, b, i, q);
      s_lo[r] = s.lo, s_hi[r] = r < rows ? s.hi : 0, s_pos[r] = s.pos;
      s_out[r] = (int)(q.q0 + i) * p.q_heads + head;
      s_slope[r] = p.slopes ? p.slopes[head] * kLog2e : 0.f;
      s_top[r] = 0;
    }
    __syncthreads();
    float v[kPasses][8];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int item = i * 128 + threadIdx.x, r = item / (NB * 4), c = item - r * (NB * 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
      if (item < kItems && r < rows) {
        const int tok = s_out[r] / p.q_heads, head = s_out[r] - tok * p.q_heads;
        const int64_t src = (int64_t)tok * p.q_st + (int64_t)head * p.q_sh + c * 8;
        load4_as(p.q, src, p.dtype, *reinterpret_cast<float(*)[4]>(&v[i][0]));
        load4_as(p.q, src + 4, p.dtype, *reinterpret_cast<float(*)[4]>(&v[i][4]));
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[i][e]));
        atomicMax(&s_top[r], __float_as_int(top));
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int item = i * 128 + threadIdx.x, r = min(item / (NB * 4), R - 1), c = item - r * (NB * 4);
      // 2^(13 - e) for a largest magnitude in [2^e, 2^(e+1)); e bounded so that the factors stay normal numbers
      const int e2 = max(-100, (s_top[r] >> 23) - 127);
      const float up = __int_as_float((127 + 13 - e2) << 23);
      float sum = 0.f;
      uint32_t w[PARTS][4];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[i][e] *= up;
        if (PARTS == 1) v[i][e] = __half2float(__float2half_rn(v[i][e]));
        sum += v[i][e];
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const int l = c & 3, k = c >> 2;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // q4_0: values 0, 2 | 1, 3 of each run of 4, the nibbles of bits 4-7 and 12-15 a 16th; q8_0: runs of 2
        float lo = FMT == 0 ? v[i][(j >> 1) * 4 + (j & 1)] : v[i][2 * j];
        float hi = FMT == 0 ? v[i][(j >> 1) * 4 + (j & 1) + 2] : v[i][2 * j + 1];
        if (FMT == 0 && l >= 2) lo *= 0.0625f, hi *= 0.0625f;
        w[0][j] = pack_half2(lo, hi);
        if constexpr (PARTS == 2) {
          const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&w[0][j]));
          w[1][j] = pack_half2(lo - back.x, hi - back.y);
        }
      }
      if (item < kItems) {
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          uint32_t* dst = reinterpret_cast<uint32_t*>(sq + (part * R + r) * NB * 4 + k * 4);
          if constexpr (FMT == 0) {  // t = 2 (l % 2) + j / 2, register 2 (j % 2) + l / 2
#pragma unroll
            for (int j = 0; j < 4; ++j) dst[(2 * (l & 1) + (j >> 1)) * 4 + 2 * (j & 1) + (l >> 1)] = w[part][j];
          } else {
            sq[(part * R + r) * NB * 4 + k * 4 + l] = make_uint4(w[part][0], w[part][1], w[part][2], w[part][3]);
          }
        }
        if (l == 0) s_start[r * NB + k] = sum * (-kOff * 0x1p-24f);
        if (c == 0) {
          float f = __int_as_float((127 + e2 - 13) << 23) * p.scale * (SIGNED ? 1.f : 0x1p24f);
          f *= p.softcap > 0.f ? 1.f / p.softcap : kLog2e;
          // a positive number always: masked scores are -inf times it, and a row of zeros has scores of 0 (what passes f32
          // here are scales for which scores are 0, or equal to the largest alone, either way)
          s_rowf[r] = fminf(fmaxf(f, FLT_MIN), FLT_MAX);
        }
      }
    }
    __syncthreads();
    uint4 qb[NT][NB][PARTS];
    float start[NT][NB][2], mul[NT][2];  // mul: scores to exponents of 2 (1 where they are that already)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < NB; ++k) {
#pragma unroll
        for (int part = 0; part < PARTS; ++part) qb[nt][k][part] = sq[(part * R + nt * 8 + g) * NB * 4 + k * 4 + t];
#pragma unroll
        for (int c = 0; c < 2; ++c)
          start[nt][k][c] = SIGNED ? 0.f : s_start[(nt * 8 + 2 * t + c) * NB + k];
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) mul[nt][c] = special ? 1.f : s_rowf[nt * 8 + 2 * t + c];
    }
    int all_lo = 0, all_hi = INT_MAX;  // keys that every row sees: no mask
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (r < rows) all_lo = max(all_lo, s_lo[r]), all_hi = min(all_hi, s_hi[r]);
    __syncthreads();  // the operands are read: the last stage may fill
    copy(begin + warp + (S - 1) * W, S - 1, ids[S - 1]);
    int id = page_of(begin + warp + S * W);

    float o[NT][NB][2][4], ref[NT][2], sum[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      ref[nt][0] = ref[nt][1] = kNoRef;
      sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int m = 0; m < 2; ++m) o[nt][k][m][0] = o[nt][k][m][1] = o[nt][k][m][2] = o[nt][k][m][3] = 0.f;
    }

    int slot = 0;
    for (int st = begin + warp; st < stop; st += W) {
      cp_async_wait<S - 1>();
      __syncwarp();
      const uint8_t* base = ring + slot * (W * C::kStage);
      const uint8_t* kscales = base + 2 * C::kQuants;
      const uint8_t* vscales = kscales + C::kScales;
      uint32_t here = 0;
#pragma unroll
      for (int s = 0; s < S; ++s) here = s == slot ? good[s] : here;
      const bool whole = st * STG >= all_lo && st * STG + STG <= all_hi && here == full;

      // UN sub-tiles of 16 keys at a time: their chains of dependent instructions overlap. Twice: with (careful) and
      // without what only some calls and a sequence's ends need, so that the common loop is short and runs straight on.
      auto steps = [&](auto careful) {
        float rowf[NT][2], slope[NT][2];
        int where[NT][2];
        if (careful.value && special) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int r = nt * 8 + 2 * t + c;
              rowf[nt][c] = s_rowf[r], slope[nt][c] = s_slope[r], where[nt][c] = s_pos[r] - st * STG - tokA;
            }
        }
#pragma unroll 1
      for (int u0 = 0; u0 < SUB; u0 += UN) {
        // ---- scores
        float x[UN][NT][4];
        float dA[UN][NB], dB[UN][NB];
#pragma unroll
        for (int i = 0; i < UN; ++i) {
          const int rowA = (u0 + i) * 16 + tokA;
          lds_scales<NB>(kscales + rowA * NB * 2, dA[i]);
          lds_scales<NB>(kscales + (rowA + 8) * NB * 2, dB[i]);
          constexpr int KW = FMT == 0 ? NB : 2 * NB;
          uint32_t wA[KW], wB[KW];
          lds_words<KW>(base + rowA * C::kRow + t * KW * 4, wA);
          lds_words<KW>(base + (rowA + 8) * C::kRow + t * KW * 4, wB);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) x[i][nt][0] = x[i][nt][1] = x[i][nt][2] = x[i][nt][3] = 0.f;
#pragma unroll
          for (int k = 0; k < NB; ++k) {
            uint32_t a[2][4];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              if constexpr (FMT == 0) {
                a[s][0] = low_nibbles<SIGNED>(wA[k] >> (8 * s)), a[s][1] = low_nibbles<SIGNED>(wB[k] >> (8 * s));
                a[s][2] = high_nibbles<SIGNED>(wA[k] >> (8 * s)), a[s][3] = high_nibbles<SIGNED>(wB[k] >> (8 * s));
              } else {
                a[s][0] = two_bytes<SIGNED>(wA[2 * k + s], 0), a[s][1] = two_bytes<SIGNED>(wB[2 * k + s], 0);
                a[s][2] = two_bytes<SIGNED>(wA[2 * k + s], 1), a[s][3] = two_bytes<SIGNED>(wB[2 * k + s], 1);
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float c[4];
              mma_16816(c, a[0][0], a[0][1], a[0][2], a[0][3], qb[nt][k][0].x, qb[nt][k][0].y, 0.f, 0.f, 0.f, 0.f);
              mma_16816(c, a[1][0], a[1][1], a[1][2], a[1][3], qb[nt][k][0].z, qb[nt][k][0].w);
              if constexpr (PARTS == 2) {
                mma_16816(c, a[0][0], a[0][1], a[0][2], a[0][3], qb[nt][k][1].x, qb[nt][k][1].y);
                mma_16816(c, a[1][0], a[1][1], a[1][2], a[1][3], qb[nt][k][1].z, qb[nt][k][1].w);
              }
              if constexpr (!SIGNED) {
#pragma unroll
                for (int e = 0; e < 4; ++e) c[e] += start[nt][k][e & 1];
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) x[i][nt][e] = fmaf(e < 2 ? dA[i][k] : dB[i][k], c[e], x[i][nt][e]);
            }
          }
          lds_scales<NB>(vscales + rowA * NB * 2, dA[i]);  // from here on the value scales of the lane's two tokens
          lds_scales<NB>(vscales + (rowA + 8) * NB * 2, dB[i]);
        }
        if (careful.value && special) {
          if (p.softcap > 0.f) {  // rowf makes these the cap's arguments
            float far = 0.f;
#pragma unroll
            for (int i = 0; i < UN; ++i)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  x[i][nt][e] *= rowf[nt][e & 1];
                  far = fmaxf(far, fabsf(x[i][nt][e]));
                }
            const float cap = p.softcap * kLog2e;
            const bool any_far = __any_sync(0xffffffffu, far > kTanhLimit);
#pragma unroll
            for (int i = 0; i < UN; ++i)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float z = x[i][nt][e];
                  float y = tanh_near(z);
                  if (any_far) y = fabsf(z) <= kTanhLimit ? y : tanh_far(z);
                  x[i][nt][e] = cap * y;
                }
          } else {
#pragma unroll
            for (int i = 0; i < UN; ++i)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[i][nt][e] *= rowf[nt][e & 1];
          }
          if (p.slopes) {
#pragma unroll
            for (int i = 0; i < UN; ++i)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int far = where[nt][e & 1] - (u0 + i) * 16 - (e >> 1) * 8;
                  x[i][nt][e] = fmaf(-slope[nt][e & 1], fabsf((float)far), x[i][nt][e]);
                }
          }
        }
        if (careful.value && !whole) {
#pragma unroll
          for (int i = 0; i < UN; ++i)
#pragma unroll
            for (int e2 = 0; e2 < 2; ++e2) {
              const int row = (u0 + i) * 16 + tokA + e2 * 8, j = st * STG + row;
              const bool read = (here >> (row >> piece_shift)) & 1;  // its page was read
              bool seen = false;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  const int r = nt * 8 + 2 * t + c;
                  if (!read || j < s_lo[r] || j >= s_hi[r])
                    x[i][nt][e2 * 2 + c] = -INFINITY;
                  else
                    seen = true;
                }
              // the scales of a token that no row sees must not enter; one that is not finite would reach the rows that
              // do not see it as 0 * d: it is taken off, and makes the rows that see it NaN
              float most = 0.f;
#pragma unroll
              for (int k = 0; k < NB; ++k) most = most + fabsf(e2 ? dB[i][k] : dA[i][k]);
              if (!seen || !(most < INFINITY)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int c = 0; c < 2; ++c)
                    if (x[i][nt][e2 * 2 + c] != -INFINITY) x[i][nt][e2 * 2 + c] = NAN;
#pragma unroll
                for (int k = 0; k < NB; ++k) (e2 ? dB[i][k] : dA[i][k]) = 0.f;
              }
            }
        }

        // ---- reference exponents: raised only where a weight times a value scale could pass 2^15
        // ceil(log2) of the lane's largest scale from its exponent bits, within 2^-30 (no scale) and 2^17 (an infinite
        // one, which must not lower the weights of a row that does not see it)
        float dtop = 0.f;
#pragma unroll
        for (int i = 0; i < UN; ++i)
#pragma unroll
          for (int k = 0; k < NB; ++k) dtop = fmaxf(dtop, fmaxf(fabsf(dA[i][k]), fabsf(dB[i][k])));
        const float dlog = (float)(min(max((int)(__float_as_uint(dtop) >> 23), 97), 143) - 126);
        bool raise = false;
        float top[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float m = fmaxf(x[0][nt][c], x[0][nt][2 + c]);
#pragma unroll
            for (int i = 1; i < UN; ++i) m = fmaxf(m, fmaxf(x[i][nt][c], x[i][nt][2 + c]));
            top[nt][c] = fmaf(m, mul[nt][c], dlog);
            raise |= top[nt][c] > ref[nt][c] + 15.f;
          }
        if (__builtin_expect(__any_sync(0xffffffffu, raise), 0)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float m = top[nt][c] - 8.f;
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
              if (m > ref[nt][c]) {
                const float f = exp2_approx(ref[nt][c] - m);
                ref[nt][c] = m;
                sum[nt][c] *= f;
#pragma unroll
                for (int k = 0; k < NB; ++k)
#pragma unroll
                  for (int mt = 0; mt < 2; ++mt) o[nt][k][mt][c] *= f, o[nt][k][mt][2 + c] *= f;
              }
            }
        }

        // ---- weights and values
#pragma unroll
        for (int i = 0; i < UN; ++i) {
          float w[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              w[nt][e] = exp2_approx(fmaf(x[i][nt][e], mul[nt][e & 1], -ref[nt][e & 1]));
              sum[nt][e & 1] += w[nt][e];
            }
          constexpr int VW = FMT == 0 ? (NB + 1) / 2 : NB;
          uint32_t v[4][VW];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int row = (u0 + i) * 16 + (j & 1 ? vtok1 : vtok0) + (j & 2 ? 8 : 0);
            const uint8_t* at = base + C::kQuants + row * C::kRow + g * NB * (FMT == 0 ? 2 : 4);
            if constexpr (FMT == 0)
              lds_halves<NB>(at, v[j]);
            else
              lds_words<NB>(at, v[j]);
          }
#pragma unroll
          for (int k = 0; k < NB; ++k) {
            uint32_t a[2][4];
            if constexpr (FMT == 0) {
              // the 16 bits of both tokens of a pair: values 2g, 16+2g, 2g+1, 17+2g in nibbles 0..3
              const uint32_t lo = __byte_perm(v[0][k / 2], v[1][k / 2], (k & 1) ? 0x7632 : 0x5410);
              const uint32_t hi = __byte_perm(v[2][k / 2], v[3][k / 2], (k & 1) ? 0x7632 : 0x5410);
              a[0][0] = low_nibbles<SIGNED>(lo), a[0][1] = low_nibbles<SIGNED>(lo >> 8);
              a[0][2] = low_nibbles<SIGNED>(hi), a[0][3] = low_nibbles<SIGNED>(hi >> 8);
              a[1][0] = high_nibbles<SIGNED>(lo), a[1][1] = high_nibbles<SIGNED>(lo >> 8);
              a[1][2] = high_nibbles<SIGNED>(hi), a[1][3] = high_nibbles<SIGNED>(hi >> 8);
            } else {
              // bytes i of both tokens of a pair: values 4g + i
#pragma unroll
              for (int mt = 0; mt < 2; ++mt) {
                const uint32_t lo = __byte_perm(v[0][k], v[1][k], mt ? 0x7362 : 0x5140);
                const uint32_t hi = __byte_perm(v[2][k], v[3][k], mt ? 0x7362 : 0x5140);
                a[mt][0] = two_bytes<SIGNED>(lo, 0), a[mt][1] = two_bytes<SIGNED>(lo, 1);
                a[mt][2] = two_bytes<SIGNED>(hi, 0), a[mt][3] = two_bytes<SIGNED>(hi, 1);
              }
            }
            if constexpr (!SIGNED) {  // less the offset, still as subnormals: values cancel in no sum
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                a[0][j] = add_half2(a[0][j], FMT == 0 ? 0x80088008u : 0x80808080u);
                a[1][j] = add_half2(a[1][j], 0x80808080u);
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float y[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) y[e] = w[nt][e] * (e < 2 ? dA[i][k] : dB[i][k]);
              const uint32_t p0 = pack_half2(y[0], y[1]), p1 = pack_half2(y[2], y[3]);
              const uint32_t b0 = transpose_8x8(p0), b1 = transpose_8x8(p1);
              if constexpr (PARTS == 1) {
                mma_16816(o[nt][k][0], a[0][0], a[0][1], a[0][2], a[0][3], b0, b1);
                mma_16816(o[nt][k][1], a[1][0], a[1][1], a[1][2], a[1][3], b0, b1);
              } else {
                // the tensor cores cut their sums off (towards zero), which adds up over a long row: for f32 each
                // tile's products are summed from zero and added to the row by rounded additions
                const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&p0));
                const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&p1));
                const uint32_t l0 = transpose_8x8(pack_half2(y[0] - f0.x, y[1] - f0.y));
                const uint32_t l1 = transpose_8x8(pack_half2(y[2] - f1.x, y[3] - f1.y));
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                  float c[4];
                  mma_16816(c, a[mt][0], a[mt][1], a[mt][2], a[mt][3], l0, l1, 0.f, 0.f, 0.f, 0.f);
                  mma_16816(c, a[mt][0], a[mt][1], a[mt][2], a[mt][3], b0, b1);
#pragma unroll
                  for (int e = 0; e < 4; ++e) o[nt][k][mt][e] += c[e];
                }
              }
            }
          }
        }
      }
      };
      if (whole && !special)
        steps(std::false_type{});
      else
        steps(std::true_type{});

      // ---- the stage is read: refill it
      __syncwarp();
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (s == slot) good[s] = __ballot_sync(0xffffffffu, id >= 0);
      copy(st + S * W, slot, id);
      id = page_of(st + (S + 1) * W);
      if (++slot == S) slot = 0;
    }

    // -------------------------------------------------------------- join the warps (in the ring's memory: all is read)
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem);              // [W][R][D]
    float2* sm = reinterpret_cast<float2*>(so + W * R * D);  // [W][R] reference, sum
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float l = sum[nt][c];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int r = nt * 8 + 2 * t + c;
        if (g == 0) sm[warp * R + r] = make_float2(ref[nt][c], l);
        float* dst = so + (warp * R + r) * D + (FMT == 0 ? 2 : 4) * g;
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            const float f = (FMT == 0 && mt ? 0.0625f : 1.f) * (SIGNED ? 1.f : 0x1p24f);  // the operands' unit
            *reinterpret_cast<float2*>(dst + 32 * k + (FMT == 0 ? 16 : 2) * mt) =
                make_float2(o[nt][k][mt][c] * f, o[nt][k][mt][2 + c] * f);
          }
      }
    __syncthreads();
    const bool begun = from > 0, done = to == span.count;
    const int part = 2 * (int)blockIdx.x + (begun ? 0 : 1);  // a share ends at most one tile and begins one at most
    for (int i = threadIdx.x; i < min(rows, R) * (D / 4); i += 128) {
      const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
      float top = kNoRef, l = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, sm[w * R + r].x);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float2 m = sm[w * R + r];
        const float f = exp2_approx(m.x - top);
        const float4 z = *reinterpret_cast<const float4*>(so + (w * R + r) * D + c);
        l = fmaf(m.y, f, l);
        y[0] = fmaf(z.x, f, y[0]), y[1] = fmaf(z.y, f, y[1]), y[2] = fmaf(z.z, f, y[2]), y[3] = fmaf(z.w, f, y[3]);
      }
      if (!begun && done) {
        const float inv = l > 0.f || l != l ? __fdividef(1.f, l) : 0.f;
        store4_as(p.out, (int64_t)s_out[r] * D + c, p.dtype, y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
        if (p.lse && c == 0) p.lse[s_out[r]] = (top + log2f(l)) * kLn2;
      } else {
        store4(p.part_o + ((int64_t)part * R + r) * D + c, y[0], y[1], y[2], y[3]);
        if (c == 0) p.part_m[part * R + r] = make_float2(top, l);
      }
    }
    if (begun && done && threadIdx.x == 0) {  // this CTA ends a tile that others began: the joining kernel's work
      join.first = (int)((pos - skip + kCost) / per);
      join.rows = min(rows, R), join.row0 = rt * R, join.head0 = h * p.group, join.q0 = (int)q.q0;
    }
    pos += take, skip += take;
    if (skip == units) skip = 0, ++h;
    __syncthreads();
  }
  if (threadIdx.x == 0) p.joins[blockIdx.x] = join;
}

// Joins the parts of tiles that several CTAs worked on: CTAs (c, y) for each CTA c that ended such a tile, a warp a row at
// a time, its lanes over the dimension. The CTA that began the tile left its second part, the others their first.
template <int NB, int R>
__global__ void __launch_bounds__(128) attention_join_kernel(const AttnParams p) {
  constexpr int D = NB * 32;
  pdl_wait_then_trigger();
  const int cta = blockIdx.x, lane = threadIdx.x & 31;
  const AttnJoin join = p.joins[cta];
  if (join.first < 0) return;
  for (int r = blockIdx.y * 4 + (threadIdx.x >> 5); r < join.rows; r += gridDim.y * 4) {
    const int rr = join.row0 + r, qi = p.cu_q ? rr / p.group : 0;
    const int64_t out_row = (int64_t)(join.q0 + qi) * p.q_heads + join.head0 + (rr - qi * p.group);
    const int n = cta - join.first + 1;
    auto part_of = [&](int i) { return (int64_t)(2 * (join.first + i) + (i == 0 ? 1 : 0)) * R + r; };
    float top = kNoRef, l = 0.f, y[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) y[i] = 0.f;
    for (int i0 = 0; i0 < n; i0 += 32) {  // 32 parts at a time: a lane holds the reference and sum of one
      const int m = min(32, n - i0);
      const float2 v = lane < m ? p.part_m[part_of(i0 + lane)] : make_float2(kNoRef, 0.f);
      float now = fmaxf(top, v.x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, o));
      const float old = exp2_approx(top - now), f = lane < m ? exp2_approx(v.x - now) : 0.f;
      float s = v.y * f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      l = fmaf(l, old, s), top = now;
#pragma unroll
      for (int i = 0; i < NB; ++i) y[i] *= old;
      constexpr int kOnce = NB <= 4 ? 16 : 8;  // loads of so many parts in flight
      for (int j0 = 0; j0 < m; j0 += kOnce) {
        float z[kOnce][NB];
#pragma unroll
        for (int j = 0; j < kOnce; ++j)
#pragma unroll
          for (int c = 0; c < NB; ++c) z[j][c] = j0 + j < m ? p.part_o[part_of(i0 + j0 + j) * D + c * 32 + lane] : 0.f;
#pragma unroll
        for (int j = 0; j < kOnce; ++j) {
          const float fj = __shfl_sync(0xffffffffu, f, j0 + j);  // 0 past the last part
#pragma unroll
          for (int c = 0; c < NB; ++c) y[c] = fmaf(z[j][c], fj, y[c]);
        }
      }
    }
    const float inv = l > 0.f || l != l ? __fdividef(1.f, l) : 0.f;
#pragma unroll
    for (int i = 0; i < NB; ++i) store_elt(p.out, out_row * D + i * 32 + lane, p.dtype, y[i] * inv);
    if (p.lse && lane == 0) p.lse[out_row] = (top + log2f(l)) * kLn2;
  }
}

template <int FMT, int NB, int NT, int PARTS>
static int launch_attention_as(const AttnParams& p, int sms, int64_t max_len, cudaStream_t stream) {
  using C = KvTile<FMT, NB>;
  constexpr int kJoin = C::kWarps * NT * 8 * (NB * 32 + 2) * 4;  // the warps' results, in the ring's place
  constexpr int kSmem = C::kRing > kJoin ? C::kRing : kJoin;
  static_assert(kSmem + 2048 <= 227 * 1024, "shared memory of a CTA");
  static_assert(kv_ctas_per_sm<FMT, NB, NT, PARTS>() <= kMaxCtasPerSm, "the workspace's parts");
  auto kernel = attention_kernel<FMT, NB, NT, PARTS>;
  static std::atomic<unsigned long long> allowed{0};
  int rc = allow_smem_once(reinterpret_cast<const void*>(kernel), kSmem, allowed);
  if (rc) return rc;
  static_assert(kv_ctas_per_sm<FMT, NB, NT, PARTS>() * (kSmem + 1024 + 1024) <= 228 * 1024, "shared memory of an SM");
  const int64_t slots = (int64_t)sms * kv_ctas_per_sm<FMT, NB, NT, PARTS>();
  // no more CTAs than there can be stages; max_len bounds the lengths from above
  const int64_t most = (int64_t)p.batch * p.row_tiles * p.heads * ((max_len + C::kTokens - 1) / C::kTokens + 1);
  const int64_t ctas = most < slots ? most : slots;
  launch_maybe_pdl(kernel, dim3((unsigned)ctas), dim3(128), kSmem, stream, p);
  rc = after_launch("attention");
  if (rc) return rc;
  launch_maybe_pdl(attention_join_kernel<NB, NT * 8>, dim3((unsigned)ctas, NT * 2), dim3(128), 0, stream, p);
  return after_launch("attention_join");
}

template <int FMT>
static int launch_attention_fmt(const AttnParams& p, int dim, int rows, int sms, int64_t max_len, cudaStream_t stream) {
  const bool wide = p.dtype == B2Q_DTYPE_F32;
  auto by_rows = [&](auto nb) {
    constexpr int NB = decltype(nb)::value;
    if constexpr (NB < 8)
      if (rows == 16)
        return wide ? launch_attention_as<FMT, NB, 2, 2>(p, sms, max_len, stream) : launch_attention_as<FMT, NB, 2, 1>(p, sms, max_len, stream);
    return wide ? launch_attention_as<FMT, NB, 1, 2>(p, sms, max_len, stream) : launch_attention_as<FMT, NB, 1, 1>(p, sms, max_len, stream);
  };
  switch (dim) {
    case 64: return by_rows(std::integral_constant<int, 2>{});
    case 96: return by_rows(std::integral_constant<int, 3>{});
    case 128: return by_rows(std::integral_constant<int, 4>{});
    default: return by_rows(std::integral_constant<int, 8>{});
  }
}

}  // namespace b2q
