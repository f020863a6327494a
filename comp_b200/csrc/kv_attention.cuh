// Attention over the quantized cache for few query rows (single tokens, drafts): streams the cache once.
//
// Mathematics. For a KV head's query rows r (its query heads times the query tokens) and keys j,
//   x_rj = scale * sum_b dk_jb * (sum_{i in b} Q_ri (k_ji - off)),   o_r = sum_j 2^(x_rj log2e - ref) dv_jb (v_ji - off) / L
// in one pass, with a running reference exponent `ref` and sum L for each row. The quants are whole numbers, so both
// products run on the tensor cores (16x8x16, f16 in, f32 sums) with keys and values as the 16-row operand and 8 query
// rows as the columns: nothing is padded, and no quant is rounded. What an operand's 16 bits hold:
//   - keys: the quant's bits alone, i.e. the f16 subnormal q * 2^-24 (or q * 2^-20 for a nibble left in bits 4-7): one
//     AND unpacks two values. The offset -off * sum(Q) of a block is the sum's start value, a constant of the row.
//   - queries: scaled by a power of two to 2^13..2^14, so that 16-bit queries are exact; f32 queries take two parts.
//     A block's scale dk (per key and block) multiplies the f32 sum of the block.
//   - values: the quant minus its offset, again as an exact subnormal; no running sum can then cancel.
//   - weights: 2^(x - ref) * dv in f32 for each block, rounded once to f16 (f32 calls: two parts, 22 bits). `ref` follows
//     the row's scores and the value scales, so that the products stay at most 2^15 and a row's largest near 2^8: they
//     cannot overflow whatever the scales, and lose no bits to f16's small exponents until 2^-22 of the largest.
// A weight matrix leaves the first product with keys along the lanes' rows and enters the second with keys along their
// pairs: one 8x8 transpose in registers each.
//
// What bounds it: the cache's bytes. Every warp is on its own: it owns every W-th stage of 32 or 64 keys of its CTA's
// share, copied by its own ring of bulk copies (at most 64 keys: four contiguous pieces a page), and joins the others
// once at the end through shared memory. With few rows the keys are split over CTAs, and a second kernel joins those.
#pragma once

#include <climits>
#include <cmath>
#include <type_traits>

#include "kv_device.cuh"
#include "kv_internal.h"

namespace b2q {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNoRef = -1e30f;  // reference exponent of a row that has seen no key

template <int FMT, int NB>
struct KvTile {
  static constexpr int kRow = NB * (FMT == 0 ? 16 : 32);           // quant bytes of a token's row
  static constexpr int kTokens = kRow * 64 * 2 > 10240 ? 32 : 64;  // tokens a stage
  static constexpr int kQuants = kTokens * kRow, kScales = kTokens * NB * 2;
  static constexpr int kStage = 2 * (kQuants + kScales);
  static constexpr int kWarps = 4;
  // ring stages a warp: at most 111 KB a CTA, two CTAs an SM (one for q8_0 rows of 256)
  static constexpr int kStages = 3;
  static constexpr int kRing = kStage * kStages * kWarps;
};

// Row r of a 16-token tile is this token: chosen so that both the key loads (lanes of two rows side by side) and the
// value loads (lanes of four tokens side by side) spread over the shared-memory banks.
__device__ __forceinline__ int tile_token(int r) { return (r & 1) ? ((r >> 1) ^ 1) + 4 : (r >> 1); }

// NB consecutive 32-bit words.
template <int NB>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[NB]) {
  if constexpr (NB % 4 == 0) {
#pragma unroll
    for (int i = 0; i < NB; i += 4) {
      const uint4 v = lds_v4(addr + 4 * i);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  } else if constexpr (NB % 2 == 0) {
#pragma unroll
    for (int i = 0; i < NB; i += 2) {
      const uint2 v = lds_v2(addr + 4 * i);
      w[i] = v.x, w[i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NB; ++i) w[i] = lds_u32(addr + 4 * i);
  }
}

// NB consecutive 16-bit words, two to a register (the last register's high half is unused when NB is odd).
template <int NB>
__device__ __forceinline__ void lds_halves(uint32_t addr, uint32_t (&w)[(NB + 1) / 2]) {
  if constexpr (NB % 2 == 0) {
    lds_words<NB / 2>(addr, w);
  } else {
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const uint32_t h = lds_u16(addr + 2 * i);
      w[i / 2] = (i & 1) ? (w[i / 2] | h << 16) : h;
    }
  }
}

// The NB f16 scales of a token.
template <int NB>
__device__ __forceinline__ void lds_scales(uint32_t addr, float (&d)[NB]) {
  uint32_t w[(NB + 1) / 2];
  lds_halves<NB>(addr, w);
#pragma unroll
  for (int b = 0; b < NB; ++b) d[b] = f16_bits_to_f32((uint16_t)(w[b / 2] >> (16 * (b & 1))));
}

__device__ __forceinline__ float load_elt(const void* p, int64_t i, int dtype) {
  if (dtype == B2Q_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == B2Q_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_elt(void* p, int64_t i, int dtype, float v) {
  if (dtype == B2Q_DTYPE_F32)
    static_cast<float*>(p)[i] = v;
  else if (dtype == B2Q_DTYPE_F16)
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// cap * tanh(x / cap): an odd polynomial below 1/4 (next term under 3e-9 of it), 1 - 2 / (e^2z + 1) above.
__device__ __forceinline__ float soft_cap(float x, float cap, float inv_cap) {
  const float z = fabsf(x * inv_cap), z2 = z * z;
  const float poly = z * fmaf(z2, fmaf(z2, fmaf(z2, fmaf(z2, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
  const float far = 1.f - __fdividef(2.f, exp2_approx(z * (2.f * kLog2e)) + 1.f);
  return copysignf(cap * (z < 0.25f ? poly : far), x);
}

// The query token and head of row r of sequence b's rows for KV head h, and its visible keys.
struct QueryRow {
  int64_t token;
  int head, pos, lo, hi;
};
__device__ __forceinline__ QueryRow query_row(const AttnParams& p, int b, int h, int r, int64_t q0, int n, int len) {
  QueryRow s;
  const int i = r / p.group;
  s.head = h * p.group + (r - i * p.group);
  s.token = q0 + i;
  s.pos = len - n + i;
  s.hi = s.pos + 1;
  if (p.prefix) s.hi = max(s.hi, p.prefix[b]);
  s.hi = max(0, min(s.hi, len));
  s.lo = p.starts ? max(0, p.starts[s.token]) : 0;
  if (p.window > 0) s.lo = max(s.lo, s.pos - p.window + 1);
  return s;
}

// FMT 0 (q4_0) or 2 (q8_0), NB blocks a head, NT tiles of 8 query rows, PARTS f16 parts of queries and weights.
template <int FMT, int NB, int NT, int PARTS>
__global__ void __launch_bounds__(128) attention_kernel(const AttnParams p) {
  using C = KvTile<FMT, NB>;
  constexpr int D = NB * 32, W = C::kWarps, STG = C::kTokens, SUB = STG / 16, R = NT * 8;
  constexpr float kOff = FMT == 0 ? 8.f : 128.f;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[W * C::kStages];
  __shared__ int s_lo[R], s_hi[R], s_pos[R];
  __shared__ float s_slope[R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  int task = blockIdx.x;
  const int split = task % p.splits;
  task /= p.splits;
  const int rt = task % p.row_tiles;
  task /= p.row_tiles;
  const int h = task % p.heads, b = task / p.heads;

  const uint32_t my_bars = smem_addr(&bars[warp * C::kStages]);
  const uint32_t ring = smem_addr(smem) + warp * C::kStages * C::kStage;
  if (lane == 0) {
    for (int s = 0; s < C::kStages; ++s) mbar_init(my_bars + 8 * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait_then_trigger();

  // the sequence's query tokens, held within q whatever cu_q says
  const int64_t q0 = p.cu_q ? max((int64_t)0, min((int64_t)p.cu_q[b], p.T)) : b;
  const int n = p.cu_q ? (int)(min((int64_t)p.cu_q[b + 1], p.T) - q0) : 1;
  const int rows = n * p.group - rt * R;  // rows from this tile on
  if (rows <= 0) return;
  const int len = max(0, min(p.lens[b], p.table_pages << p.page_shift));
  if (p.lens[b] > len && threadIdx.x == 0) atomicCAS(&g_device_error, 0, kErrPage);

  // visible keys of the tile's rows: their union is read, their intersection needs no mask
  if (threadIdx.x < R) {
    const int r = threadIdx.x;
    const bool there = r < rows;
    const QueryRow s = query_row(p, b, h, rt * R + (there ? r : 0), q0, n, len);
    s_lo[r] = s.lo;
    s_hi[r] = there ? s.hi : 0;
    s_pos[r] = s.pos;
    s_slope[r] = p.slopes ? p.slopes[s.head] * kLog2e : 0.f;
  }
  __syncthreads();
  int first = INT_MAX, last = 0, all_lo = 0, all_hi = INT_MAX;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= rows) continue;
    const int lo = s_lo[r], hi = s_hi[r];
    if (lo < hi) first = min(first, lo), last = max(last, hi);
    all_lo = max(all_lo, lo), all_hi = min(all_hi, hi);
  }
  first = min(first, last) / STG;
  const int stages = (last + STG - 1) / STG - first;  // of the whole tile
  const int begin = first + (int)((int64_t)stages * split / p.splits);
  const int end = first + (int)((int64_t)stages * (split + 1) / p.splits);

  // ---------------------------------------------------------------- the ring: lane i copies piece i / 4, plane i % 4
  const uint64_t pol = evict_first_policy();
  const int page = 1 << p.page_shift;
  const int piece = min(page, STG), pieces = STG / piece;
  const int32_t* table = p.table + (int64_t)b * p.table_stride;
  const int my_piece = lane >> 2, plane = lane & 3;
  // the page of this lane's piece of a stage, or -1
  auto page_of = [&](int stage) -> int {
    const int tok = stage * STG + my_piece * piece;
    if (stage >= end || my_piece >= pieces || tok >= last) return -1;
    const int id = table[tok >> p.page_shift];
    if (id < 0 || id >= p.pages) {
      atomicCAS(&g_device_error, 0, kErrPage);
      return -1;
    }
    return id;
  };
  auto issue = [&](int stage, int slot, int id) {
    const int bytes = plane < 2 ? piece * C::kRow : piece * NB * 2;
    int total = id >= 0 ? bytes : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const uint32_t bar = my_bars + 8 * slot;
    if (lane == 0) mbar_expect_tx(bar, (uint32_t)total);
    __syncwarp();
    if (id >= 0) {
      const int off = (stage * STG + my_piece * piece) & (page - 1);
      const int64_t row = (((int64_t)id * p.heads + h) << p.page_shift) + off;
      const uint32_t base = ring + slot * C::kStage;
      if (plane == 0)
        bulk_g2s(base + my_piece * bytes, p.kq + row * C::kRow, bytes, bar, pol);
      else if (plane == 1)
        bulk_g2s(base + C::kQuants + my_piece * bytes, p.vq + row * C::kRow, bytes, bar, pol);
      else if (plane == 2)
        bulk_g2s(base + 2 * C::kQuants + my_piece * bytes, p.ks + row * NB, bytes, bar, pol);
      else
        bulk_g2s(base + 2 * C::kQuants + C::kScales + my_piece * bytes, p.vs + row * NB, bytes, bar, pol);
    }
  };
  // a page that cannot be read masks its tokens: the bits of a stage's good pieces (lane 4 * piece votes)
  uint32_t good[C::kStages];
  int ids = page_of(begin + warp);
#pragma unroll
  for (int s = 0; s < C::kStages; ++s) {
    const int st = begin + warp + s * W;
    good[s] = __ballot_sync(0xffffffffu, ids >= 0);
    if (st < end) issue(st, s, ids);
    ids = page_of(st + W);
  }

  // ---------------------------------------------------------------- queries: B operands, row scales, start values
  uint32_t qb[NT][NB][2][2][PARTS];
  float start[NT][NB][2], rowf[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = rt * R + nt * 8 + g;
    const bool there = nt * 8 + g < rows;
    const int i = r / p.group;
    const int64_t src = there ? (q0 + i) * p.q_st + (int64_t)(h * p.group + r - i * p.group) * p.q_sh : 0;
    float v[NB][8], top = 0.f;
#pragma unroll
    for (int k = 0; k < NB; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = FMT == 0 ? 32 * k + 4 * t + (e & 3) + (e >> 2) * 16 : 32 * k + 8 * t + e;
        v[k][e] = there ? load_elt(p.q, src + at, p.dtype) : 0.f;
        top = fmaxf(top, fabsf(v[k][e]));
      }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^(13 - e) for a largest magnitude in [2^e, 2^(e+1)); e bounded so that the factors stay normal numbers
    const int e2 = max(-100, (int)(__float_as_uint(top) >> 23) - 127);
    const float up = __uint_as_float((uint32_t)(127 + 13 - e2) << 23);
    float f = __uint_as_float((uint32_t)(127 + e2 - 13) << 23) * p.scale * 0x1p24f;
    if (p.softcap <= 0.f) f *= kLog2e;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float x = v[k][e] * up;
        if (PARTS == 1) x = __half2float(__float2half_rn(x));
        sum += x;
        v[k][e] = x;
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum *= -kOff * 0x1p-24f;
      start[nt][k][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
      start[nt][k][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
      // (step, half): q4_0 values s and s + 2 of the low (high) nibbles; q8_0 values 4s + 2 half and the next
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          float lo = FMT == 0 ? v[k][hf * 4 + s] : v[k][s * 4 + hf * 2];
          float hi = FMT == 0 ? v[k][hf * 4 + s + 2] : v[k][s * 4 + hf * 2 + 1];
          if (FMT == 0 && hf) lo *= 0.0625f, hi *= 0.0625f;
          const uint32_t w = pack_half2(lo, hi);
          qb[nt][k][s][hf][0] = w;
          if (PARTS == 2) {
            const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&w));
            qb[nt][k][s][hf][PARTS - 1] = pack_half2(lo - back.x, hi - back.y);
          }
        }
    }
    rowf[nt][0] = __shfl_sync(0xffffffffu, f, 8 * t);
    rowf[nt][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
  }

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
  const float inv_cap = p.softcap > 0.f ? 1.f / p.softcap : 0.f;
  const int tokA = tile_token(g);                                // key rows g and g + 8 of a tile: tokA, tokA + 8
  const int vtok0 = tile_token(2 * t), vtok1 = tile_token(2 * t + 1);

  bool ok = true;
  int slot = 0;
  uint32_t parity = 0;
  for (int st = begin + warp; st < end; st += W) {
    if (!__all_sync(0xffffffffu, mbar_wait(my_bars + 8 * slot, parity, kWaitLimit))) {
      ok = false;
      break;
    }
    const uint32_t base = ring + slot * C::kStage;
    const int j0 = st * STG;
    uint32_t here = 0;
#pragma unroll
    for (int s = 0; s < C::kStages; ++s) here = s == slot ? good[s] : here;
    const bool whole = j0 >= all_lo && j0 + STG <= all_hi && __popc(here) == 4 * pieces;

    // ---- scores
    float x[NT][SUB][4];
    float dtop = 0.f;  // largest value scale of this lane's tokens
    float dv[SUB][2][NB];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      float acc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
      const int rowA = u * 16 + tokA, rowB = rowA + 8;
      float dA[NB], dB[NB];
      lds_scales<NB>(base + 2 * C::kQuants + rowA * NB * 2, dA);
      lds_scales<NB>(base + 2 * C::kQuants + rowB * NB * 2, dB);
      constexpr int KW = FMT == 0 ? NB : 2 * NB;
      uint32_t wA[KW], wB[KW];
      lds_words<KW>(base + rowA * C::kRow + t * KW * 4, wA);
      lds_words<KW>(base + rowB * C::kRow + t * KW * 4, wB);
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        uint32_t a[2][4];
        if constexpr (FMT == 0) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            a[s][0] = (wA[k] >> (8 * s)) & 0x000f000fu, a[s][1] = (wB[k] >> (8 * s)) & 0x000f000fu;
            a[s][2] = (wA[k] >> (8 * s)) & 0x00f000f0u, a[s][3] = (wB[k] >> (8 * s)) & 0x00f000f0u;
          }
        } else {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            a[s][0] = __byte_perm(wA[2 * k + s], 0, 0x4140), a[s][1] = __byte_perm(wB[2 * k + s], 0, 0x4140);
            a[s][2] = __byte_perm(wA[2 * k + s], 0, 0x4342), a[s][3] = __byte_perm(wB[2 * k + s], 0, 0x4342);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float c[4];
          mma_16816(c, a[0][0], a[0][1], a[0][2], a[0][3], qb[nt][k][0][0][0], qb[nt][k][0][1][0], start[nt][k][0],
                    start[nt][k][1], start[nt][k][0], start[nt][k][1]);
          mma_16816(c, a[1][0], a[1][1], a[1][2], a[1][3], qb[nt][k][1][0][0], qb[nt][k][1][1][0]);
          if constexpr (PARTS == 2) {
            mma_16816(c, a[0][0], a[0][1], a[0][2], a[0][3], qb[nt][k][0][0][1], qb[nt][k][0][1][1]);
            mma_16816(c, a[1][0], a[1][1], a[1][2], a[1][3], qb[nt][k][1][0][1], qb[nt][k][1][1][1]);
          }
          acc[nt][0] = fmaf(dA[k], c[0], acc[nt][0]);
          acc[nt][1] = fmaf(dA[k], c[1], acc[nt][1]);
          acc[nt][2] = fmaf(dB[k], c[2], acc[nt][2]);
          acc[nt][3] = fmaf(dB[k], c[3], acc[nt][3]);
        }
      }
      lds_scales<NB>(base + 2 * C::kQuants + C::kScales + rowA * NB * 2, dv[u][0]);
      lds_scales<NB>(base + 2 * C::kQuants + C::kScales + rowB * NB * 2, dv[u][1]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float y = acc[nt][e] * rowf[nt][e & 1];
          if (p.softcap > 0.f) y = soft_cap(y, p.softcap, inv_cap) * kLog2e;
          x[nt][u][e] = y;
        }
      if (p.slopes) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = nt * 8 + 2 * t + (e & 1), j = j0 + rowA + (e >> 1) * 8;
            x[nt][u][e] -= s_slope[r] * (float)abs(s_pos[r] - j);
          }
      }
      if (!whole) {
#pragma unroll
        for (int e2 = 0; e2 < 2; ++e2) {
          const int j = j0 + rowA + e2 * 8;
          // pages that were not read, and tokens past the last: nothing of theirs may enter
          const bool read = (here >> (4 * ((rowA + e2 * 8) / piece))) & 1;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int r = nt * 8 + 2 * t + c;
              if (!read || j < s_lo[r] || j >= s_hi[r]) x[nt][u][e2 * 2 + c] = -INFINITY;
            }
          bool seen = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) seen |= x[nt][u][e2 * 2] != -INFINITY || x[nt][u][e2 * 2 + 1] != -INFINITY;
          if (!seen) {
#pragma unroll
            for (int k = 0; k < NB; ++k) dv[u][e2][k] = 0.f;
          }
        }
      }
#pragma unroll
      for (int k = 0; k < NB; ++k) dtop = fmaxf(dtop, fmaxf(fabsf(dv[u][0][k]), fabsf(dv[u][1][k])));
    }

    // ---- reference exponents: raised only where a weight times a value scale could pass 2^15
    // ceil(log2) of the lane's largest scale from its exponent bits, within 2^-30 (no scale) and 2^17 (an infinite one,
    // which must not lower the weights of a row that does not see it)
    const float dlog = (float)(min(max((int)(__float_as_uint(dtop) >> 23), 97), 143) - 126);
    bool raise = false;
    float top[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < SUB; ++u) m = fmaxf(m, fmaxf(x[nt][u][c], x[nt][u][2 + c]));
        top[nt][c] = m + dlog;
        raise |= top[nt][c] - ref[nt][c] > 15.f;
      }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float m = top[nt][c];
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          if (m - 8.f > ref[nt][c]) {
            const float f = exp2_approx(ref[nt][c] - (m - 8.f));
            ref[nt][c] = m - 8.f;
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
    for (int u = 0; u < SUB; ++u) {
      float w[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[nt][e] = exp2_approx(x[nt][u][e] - ref[nt][e & 1]);
          sum[nt][e & 1] += w[nt][e];
        }
      constexpr int VW = FMT == 0 ? (NB + 1) / 2 : NB;
      uint32_t v[4][VW];
      const uint32_t vb = base + C::kQuants + u * 16 * C::kRow + g * NB * (FMT == 0 ? 2 : 4);
      if constexpr (FMT == 0) {
        lds_halves<NB>(vb + vtok0 * C::kRow, v[0]);
        lds_halves<NB>(vb + vtok1 * C::kRow, v[1]);
        lds_halves<NB>(vb + (vtok0 + 8) * C::kRow, v[2]);
        lds_halves<NB>(vb + (vtok1 + 8) * C::kRow, v[3]);
      } else {
        lds_words<NB>(vb + vtok0 * C::kRow, v[0]);
        lds_words<NB>(vb + vtok1 * C::kRow, v[1]);
        lds_words<NB>(vb + (vtok0 + 8) * C::kRow, v[2]);
        lds_words<NB>(vb + (vtok1 + 8) * C::kRow, v[3]);
      }
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        uint32_t a[2][4];
        if constexpr (FMT == 0) {
          // the 16 bits of both tokens of a pair: values 2g, 16+2g, 2g+1, 17+2g in nibbles 0..3
          const uint32_t lo = __byte_perm(v[0][k / 2], v[1][k / 2], (k & 1) ? 0x7632 : 0x5410);
          const uint32_t hi = __byte_perm(v[2][k / 2], v[3][k / 2], (k & 1) ? 0x7632 : 0x5410);
          a[0][0] = add_half2(lo & 0x000f000fu, 0x80088008u), a[0][1] = add_half2((lo >> 8) & 0x000f000fu, 0x80088008u);
          a[0][2] = add_half2(hi & 0x000f000fu, 0x80088008u), a[0][3] = add_half2((hi >> 8) & 0x000f000fu, 0x80088008u);
          a[1][0] = add_half2(lo & 0x00f000f0u, 0x80808080u), a[1][1] = add_half2((lo >> 8) & 0x00f000f0u, 0x80808080u);
          a[1][2] = add_half2(hi & 0x00f000f0u, 0x80808080u), a[1][3] = add_half2((hi >> 8) & 0x00f000f0u, 0x80808080u);
        } else {
          // bytes i of both tokens of a pair: values 4g + i
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            const uint32_t lo = __byte_perm(v[0][k], v[1][k], mt ? 0x7362 : 0x5140);
            const uint32_t hi = __byte_perm(v[2][k], v[3][k], mt ? 0x7362 : 0x5140);
            a[mt][0] = add_half2(__byte_perm(lo, 0, 0x4140), 0x80808080u);
            a[mt][1] = add_half2(__byte_perm(lo, 0, 0x4342), 0x80808080u);
            a[mt][2] = add_half2(__byte_perm(hi, 0, 0x4140), 0x80808080u);
            a[mt][3] = add_half2(__byte_perm(hi, 0, 0x4342), 0x80808080u);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = w[nt][e] * dv[u][e >> 1][k];
          if (!whole) {  // a masked key's scale may be anything
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = x[nt][u][e] == -INFINITY ? 0.f : y[e];
          }
          const uint32_t p0 = pack_half2(y[0], y[1]), p1 = pack_half2(y[2], y[3]);
          const uint32_t b0 = transpose_8x8(p0), b1 = transpose_8x8(p1);
          mma_16816(o[nt][k][0], a[0][0], a[0][1], a[0][2], a[0][3], b0, b1);
          mma_16816(o[nt][k][1], a[1][0], a[1][1], a[1][2], a[1][3], b0, b1);
          if constexpr (PARTS == 2) {
            const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&p0));
            const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&p1));
            const uint32_t l0 = transpose_8x8(pack_half2(y[0] - f0.x, y[1] - f0.y));
            const uint32_t l1 = transpose_8x8(pack_half2(y[2] - f1.x, y[3] - f1.y));
            mma_16816(o[nt][k][0], a[0][0], a[0][1], a[0][2], a[0][3], l0, l1);
            mma_16816(o[nt][k][1], a[1][0], a[1][1], a[1][2], a[1][3], l0, l1);
          }
        }
      }
    }

    // ---- the stage is read: refill it
    __syncwarp();
    const int next = st + C::kStages * W;
    const uint32_t vote = __ballot_sync(0xffffffffu, ids >= 0);
#pragma unroll
    for (int s = 0; s < C::kStages; ++s)
      if (s == slot) good[s] = vote;
    if (next < end) issue(next, slot, ids);
    ids = page_of(next + W);
    if (++slot == C::kStages) slot = 0, parity ^= 1;
  }
  if (!ok && lane == 0) atomicCAS(&g_device_error, 0, kErrTimeout);

  // ---------------------------------------------------------------- join the warps
  // every copy that was issued has been waited for (a wait that gave up returns with its copies drained below)
  if (!ok) {
    for (int s = 0; s < C::kStages; ++s) mbar_wait(my_bars + 8 * s, 0, kWaitLimit), mbar_wait(my_bars + 8 * s, 1, kWaitLimit);
  }
  __syncthreads();  // the ring's memory is free
  float* so = reinterpret_cast<float*>(smem);                    // [W][R][D]
  float2* sm = reinterpret_cast<float2*>(so + W * R * D);        // [W][R] reference, sum
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float l = sum[nt][c];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const int r = nt * 8 + 2 * t + c;
      if (g == 0) sm[warp * R + r] = make_float2(ok ? ref[nt][c] : NAN, l);
      float* dst = so + (warp * R + r) * D;
#pragma unroll
      for (int k = 0; k < NB; ++k)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const float f = FMT == 0 && mt ? 0x1p20f : 0x1p24f;  // the unit of the quants' bits
          const int at = FMT == 0 ? 32 * k + 16 * mt + 2 * g : 32 * k + 4 * g + 2 * mt;
          dst[at] = o[nt][k][mt][c] * f;
          dst[at + 1] = o[nt][k][mt][2 + c] * f;
        }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < R * D; i += 128) {
    const int r = i / D, c = i - r * D;
    if (r >= rows) break;
    float m = kNoRef;
    bool bad = false;
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, sm[w * R + r].x), bad |= isnan(sm[w * R + r].x);
    float l = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float2 v = sm[w * R + r];
      const float f = bad ? NAN : exp2_approx(v.x - m);
      l += v.y * f;
      y += so[(w * R + r) * D + c] * f;
    }
    const int rr = rt * R + r, qi = rr / p.group;
    const int64_t out_row = (q0 + qi) * p.q_heads + h * p.group + (rr - qi * p.group);
    if (p.splits == 1) {
      store_elt(p.out, out_row * D + c, p.dtype, l > 0.f || l != l ? y / l : 0.f);
      if (p.lse && c == 0) p.lse[out_row] = (m + log2f(l)) * kLn2;
    } else {
      p.part_o[(out_row * p.splits + split) * D + c] = y;
      if (c == 0) p.part_m[out_row * p.splits + split] = make_float2(m, l);
    }
  }
}

template <int FMT, int NB, int NT, int PARTS>
static int launch_attention_as(const AttnParams& p, cudaStream_t stream) {
  using C = KvTile<FMT, NB>;
  constexpr int kJoin = C::kWarps * NT * 8 * (NB * 32 + 2) * 4;
  constexpr int kSmem = C::kRing > kJoin ? C::kRing : kJoin;
  static_assert(kSmem + 2048 <= 227 * 1024, "shared memory of a CTA");
  auto kernel = attention_kernel<FMT, NB, NT, PARTS>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return fail(B2Q_ECUDA, "b2q_attention: %s", cudaGetErrorString(e));
  const int64_t ctas = (int64_t)p.batch * p.heads * p.row_tiles * p.splits;
  launch_maybe_pdl(kernel, dim3((unsigned)ctas), dim3(128), kSmem, stream, p);
  return after_launch("attention");
}

template <int FMT>
static int launch_attention_fmt(const AttnParams& p, int dim, int rows, cudaStream_t stream) {
  const bool wide = p.dtype == B2Q_DTYPE_F32;
  auto by_rows = [&](auto nb) {
    constexpr int NB = decltype(nb)::value;
    if constexpr (NB < 8)
      if (rows == 16)
        return wide ? launch_attention_as<FMT, NB, 2, 2>(p, stream) : launch_attention_as<FMT, NB, 2, 1>(p, stream);
    return wide ? launch_attention_as<FMT, NB, 1, 2>(p, stream) : launch_attention_as<FMT, NB, 1, 1>(p, stream);
  };
  switch (dim) {
    case 64: return by_rows(std::integral_constant<int, 2>{});
    case 96: return by_rows(std::integral_constant<int, 3>{});
    case 128: return by_rows(std::integral_constant<int, 4>{});
    default: return by_rows(std::integral_constant<int, 8>{});
  }
}

}  // namespace b2q
