// Attention over the quantized cache for many query rows (prompt chunks): the fifth-generation tensor cores.
//
// A CTA works on up to 256 rows (two tiles of 128) of one KV head against blocks of 128 keys. Four roles:
//   - a warpgroup unpacks the block's keys and values to f16 once for all rows, into tiles of core matrices (8 rows of 16
//     bytes, K-major, no swizzle): keys as [8 values of a key][key], values transposed, as [8 keys of a column][column];
//   - one thread issues the products: S = Q K^T into tensor memory, and O += P V with P read from tensor memory;
//   - two warpgroups, a row a thread, turn S into P (f16, in S's own columns) and keep the row's reference exponent and
//     sum in f32; the other tile's products run meanwhile. The reference lies 2^7 below the row's maximum
//     (so that f16 holds small weights) and follows it only when that has grown by more than 2^8: then the thread rescales
//     its row of O, which no product is using at that time.
// Queries are scaled by a power of two a row, its largest to 2^6 (exact for f16 values down to 2^-20 of that and bf16 values
// down to 2^-23, the others within 2^-31 of it), and take the order of the keys' packed words, so that one word of a key
// becomes one 16-byte chunk of its operand. Values are rounded to f16 (11 bits), and so are keys and weights for bf16 calls,
// whose outputs' own rounding (8 bits) is far larger; for f16 calls, where it is not, both enter in two parts (22 bits; error
// against 64 bits 1.3 to 1.4 times one rounding's, in one part 1.6 to 2.6). A key with values past f16's range (65504) enters
// its operand a power of two smaller, and its scores, or its weights, are made as much larger: passes of their own over such
// a block, as for keys without a page, which are masked.
//
// What bounds it: 128 keys for 256 rows of 128 values take 2048 cycles on the tensor cores, 2048 on the units that compute
// 2^x (16 a cycle), and about 2048 of shared memory's (operands of S from there twice, unpacked tiles into it); a tile's
// chain - S, softmax, P V - is longer than the other tile's products that run beside it. Measured: a chunk of 2048 queries
// at the end of 32768 keys, 32 heads on 8 of 128, bf16: 1.22 ms in a long run, 874 TFLOP/s (1.11 ms at best); the softmax of
// a tile takes 1.5 us a block and waits 0.8 us. What did not help: a part of the 2^x as polynomials (3 to 17% slower for an
// eighth to a half), loads of S ahead of their use (1%), one pass with the weights kept in registers (65%: they spill).
#pragma once

#include "kv_attention.cuh"

namespace b2q {

// EXACT: the scores from keys in two f16 parts, what f16 calls and calls that return lse need: one part's rounding is 1e-4
// of a score, which a bf16 output does not show, but an f16 one does, and an f32 lse (1e-5 of it; with two parts 1e-7).
// WIDE (f16 calls): the weights in two parts too, the second beside the first in S's columns. Measured in one part / in two,
// us, 32 heads on 8 of 128: four f16 prompts of 2048 281 / 346 (with lse 315 / 347), 1024 x 16384 over q8_0 355 / 440, packed
// documents 138 / 146; heads of 256, whose key parts take turns in one tile, 1024 x 8192 264 / 438.
template <int FMT, int NB, bool EXACT>
struct TcTile {
  static constexpr int D = NB * 32;
  static constexpr int kRow = NB * (FMT == 0 ? 16 : 32);  // quant bytes of a token's row
  static constexpr int MT = NB == 8 ? 1 : 2;              // row tiles: tensor memory holds O (D) and S (128) of each
  static constexpr int kBufs = NB == 8 ? 1 : 2;           // value tiles in shared memory
  // key tiles, the parts of a key, and how many of them take turns in one tile (heads of 256: no room for both)
  static constexpr int kKeyBufs = EXACT ? 1 : kBufs, kParts = EXACT ? 2 : 1, kTurns = EXACT && NB == 8 ? 2 : 1;
  static constexpr int kRows = MT * 128, kKeys = 128;
  static constexpr int kQ = 128 * D * 2, kTile = 128 * D * 2;
  static constexpr int kHeld = kKeyBufs * kParts / kTurns;  // key tiles in shared memory
  static constexpr int kSmem = MT * kQ + (kHeld + kBufs) * kTile;
  // 4 unpacking, then 1 issuing; with two row tiles three more, which only hand their registers on
  static constexpr int kSoftmaxWarps = MT * 4, kWarps = MT == 2 ? 16 : MT * 4 + 5;
  // registers of a thread at launch and after the split: 2 x 128 x 152 + 128 x 128 + 128 x 80 = 512 x 128
  static constexpr int kLaunchRegs = 128, kSoftmaxRegs = 152, kIssueRegs = 80;
  static_assert(MT == 1 || 256 * kSoftmaxRegs + 128 * kLaunchRegs + 128 * kIssueRegs <= 512 * kLaunchRegs, "registers");
  static constexpr uint32_t kS = 256;                     // column of S (and P) of tile 0; O is at 0
  // the largest scale (f16 bits) whose values all fit f16: 8 * 8188 and 128 * 511.75 are 65504; and by what power of two a
  // key or value row with a larger one is less in its operand
  static constexpr uint32_t kMost = FMT == 0 ? 0x6fffu : 0x5fffu;
  static constexpr int kLess = FMT == 0 ? 4 : 8;
};

namespace tc {

// K-major, no swizzle: the next 16 bytes of K are `lbo` bytes on, the next 8 rows 128
__device__ __forceinline__ uint64_t smem_desc_kmajor(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) |
         ((uint64_t)1 << 46);
}
// kind::f16: f32 accumulator, A and B f16, both K-major, M = 128, N = n
__device__ __forceinline__ uint32_t instr_desc_f16(int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc));
}
#define B2Q_R8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), \
                     "=r"(v[i + 6]), "=r"(v[i + 7])
#define B2Q_I8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), \
                     "r"(v[i + 6]), "r"(v[i + 7])
#define B2Q_RW8(v, i) "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3]), "+r"(v[i + 4]), "+r"(v[i + 5]), \
                      "+r"(v[i + 6]), "+r"(v[i + 7])
// 32 consecutive columns of this thread's lane, without waiting
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : B2Q_R8(v, 0), B2Q_R8(v, 8), B2Q_R8(v, 16), B2Q_R8(v, 24)
      : "r"(taddr));
}
// tcgen05.wait::ld that names the registers of a load, so that no use of them is scheduled above it
__device__ __forceinline__ void tmem_wait_ld32(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : B2Q_RW8(v, 0), B2Q_RW8(v, 8), B2Q_RW8(v, 16), B2Q_RW8(v, 24)
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::B2Q_I8(v, 0),
      B2Q_I8(v, 8), B2Q_I8(v, 16), B2Q_I8(v, 24), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::B2Q_I8(
          v, 0),
      B2Q_I8(v, 8), "r"(taddr)
      : "memory");
}
#undef B2Q_R8
#undef B2Q_I8
#undef B2Q_RW8

__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// generic writes to shared memory before the tensor cores' reads of it
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

}  // namespace tc

__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t fma_half2(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                            *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&h);
}
// (1024 + 16 q) / 16 - 72 = q - 8
__device__ __forceinline__ uint32_t high_nibbles_int(uint32_t w) {
  return fma_half2((w & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd480d480u);
}

// The largest magnitude of N f16 numbers, two to a register (an odd N's last half is 0), as f16 bits.
template <int N>
__device__ __forceinline__ uint32_t largest_half(const uint32_t (&w)[(N + 1) / 2]) {
  uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
  for (int i = 1; i < (N + 1) / 2; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  return max(m & 0xffffu, m >> 16);
}

// N bytes (a multiple of 2) of global memory into 32-bit words; 16, 8, 4 or 2 at a time as N allows (N aligned).
template <int N>
__device__ __forceinline__ void ldg_bytes(const uint8_t* at, uint32_t (&w)[(N + 3) / 4]) {
  if constexpr (N % 16 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 16) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(at + i));
      w[i / 4] = v.x, w[i / 4 + 1] = v.y, w[i / 4 + 2] = v.z, w[i / 4 + 3] = v.w;
    }
  } else if constexpr (N % 8 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(at + i));
      w[i / 4] = v.x, w[i / 4 + 1] = v.y;
    }
  } else if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) w[i / 4] = __ldg(reinterpret_cast<const uint32_t*>(at + i));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint32_t v = __ldg(reinterpret_cast<const uint16_t*>(at + i));
      w[i / 4] = (i & 2) ? (w[i / 4] | v << 16) : v;
    }
  }
}

// What beginning a tile costs a CTA, in blocks of 128 keys (as kTileCost), which take longer with a cap or a bias by
// distance. Measured with costs of 2 / 3 / 4 / 5 / 6 / 8, us, 32 heads on 8 of 128: four fresh prompts of 2048 tokens 378 /
// 320 / 298 / 278 / 276 / 282, with a cap 414 / 363 / 370 / 378 / 384 / 394; 16 ragged chunks of 32 to 300 tokens on 300 to
// 6000 keys 316 / 302 / 280 / 254 / 253 / 261, with a cap 391 / 367 / 365 / 365 / 370 / 386; documents of 500 tokens with lse
// 236 / 233 / 229 / 234 / 233 / 240, with a cap too 259 / 264 / 265 / 272 / 273 / 282.
static inline int tc_tile_cost(const AttnParams& p) { return p.softcap > 0.f || p.slopes ? 3 : 5; }

template <int FMT, int NB, bool EXACT, bool WIDE>
__global__ void __launch_bounds__(TcTile<FMT, NB, EXACT>::kWarps * 32, 1) attention_tc_kernel(const AttnParams p) {
  using C = TcTile<FMT, NB, EXACT>;
  constexpr int D = C::D, MT = C::MT, KB = C::kKeyBufs, VB = C::kBufs, TURNS = C::kTurns, R = C::kRows, STG = C::kKeys, SW = C::kSoftmaxWarps;
  extern __shared__ __align__(128) uint8_t smem[];  // queries [MT], keys [KB][parts side by side], values [VB]
  __shared__ uint64_t b_kfull[KB], b_kempty[KB], b_vfull[VB], b_vempty[VB], b_s[MT], b_p[MT], b_o[MT], b_q, b_end;
  // A block's odd keys, a bit each: those without a page, and those whose keys or whose values (s_less, written where a word
  // of s_odd is not 0) are 2^kLess less in their operands. The unpacking warps write a block's words before they hand its
  // keys on; the issuing thread, which waits for the keys, passes that on to the softmax with its own arrival at b_s. Four in
  // turn: the words of block b are written when the scores of block b - KB have ended, so when the softmax is done with
  // b - KB - 1.
  __shared__ __align__(16) uint32_t s_odd[4][STG / 32];
  __shared__ uint32_t s_less[4][2][STG / 32];
  static_assert(KB < 4, "words in turn");
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ ShareScratch<C::kWarps> plan;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // The next kernel may start only once this CTA has its tensor memory: one that took tensor memory first and then waited
  // for this grid would leave both waiting.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Share share = plan_share<STG, R, C::kWarps>(p, p.tile_cost, 1, plan);
  if (share.pos >= share.end) {
    if (threadIdx.x == 0) p.joins[blockIdx.x].first = -1;
    return;
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s_tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < KB; ++i) mbar_init(smem_addr(&b_kfull[i]), 128), mbar_init(smem_addr(&b_kempty[i]), 1);
    for (int i = 0; i < VB; ++i) mbar_init(smem_addr(&b_vfull[i]), 128), mbar_init(smem_addr(&b_vempty[i]), 1);
    for (int i = 0; i < MT; ++i) {
      mbar_init(smem_addr(&b_s[i]), 2), mbar_init(smem_addr(&b_p[i]), 128), mbar_init(smem_addr(&b_o[i]), 1);
    }
    mbar_init(smem_addr(&b_q), SW * 32), mbar_init(smem_addr(&b_end), 1);
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = s_tmem;
  const uint32_t q_smem = smem_addr(smem), k_smem = q_smem + MT * C::kQ, v_smem = k_smem + C::kHeld * C::kTile;
  // a wait that ran out ends the role's work, and the kernel at the end of the tile: every later wait is skipped
  bool ok = true;
  auto wait_one = [&](uint64_t* bar, uint32_t phase) {  // by one thread
    if (ok && !mbar_wait(smem_addr(bar), phase & 1, kWaitLimit)) ok = false, atomicExch(&s_abort, 1);
    return ok;
  };
  auto wait = [&](uint64_t* bar, uint32_t phase) {  // by a whole warp, which goes on or stops as one
    if (ok) {
      ok = __all_sync(0xffffffffu, mbar_wait(smem_addr(bar), phase & 1, kWaitLimit));
      if (!ok) atomicExch(&s_abort, 1);
    }
    return ok;
  };

  // Each role runs through the share's tiles in code of its own, so that the registers it is given are its own too.
  auto work = [&](auto role) {
    constexpr int ROLE = decltype(role)::value;  // 0 softmax, 1 unpacking, 2 issuing
  int64_t pos = share.pos;
  int entry = share.entry, h = share.head, skip = share.skip;
  AttnJoin join = {-1, 0, 0, 0, 0};
  uint32_t blocks = 0, done_tiles[2] = {0, 0}, done_blocks[2] = {0, 0}, segments = 0;  // so far: the barriers' phases
  while (pos < share.end) {
    // -------------------------------------------------------------- the next tile of the share, as in the other kernel
    const int b = p.row_tiles == 1 ? entry : entry / p.row_tiles, rt = entry - b * p.row_tiles;
    const Span span = tile_span<STG, R, true>(p, b, rt);
    if (h == p.heads || span.count == 0) {
      ++entry, h = 0;
      continue;
    }
    const int units = tile_units(span, p.tile_cost), take = (int)min((int64_t)(units - skip), share.end - pos);
    const int from = max(0, skip - p.tile_cost), to = max(0, skip + take - p.tile_cost);
    if (to == from) {
      pos += take, skip += take;
      if (skip == units) skip = 0, ++h;
      continue;
    }
    const Sequence q = sequence(p, b);
    const int rows = q.n * p.group - rt * R;  // rows from this tile on (at least 1)
    if (threadIdx.x == 0 && (q.end > q.len || (rt + 1 == p.row_tiles && rows > R)))
      atomicCAS(&g_device_error, 0, q.end > q.len ? kErrPage : kErrQueries);
    const int begin = span.first + from, n = to - from, tiles = MT == 1 || rows <= 128 ? 1 : 2;

    if constexpr (ROLE == 0) {
      // ------------------------------------------------------------ softmax: a thread owns a row
      const int tile = warp >> 2, r = tile * 128 + (warp & 3) * 32 + lane, rr = rt * R + r;
      const bool there = r < rows;
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t col_s = tmem + lanes + C::kS + tile * 128, col_o = tmem + lanes + tile * 128;
      int lo = 0, hi = INT_MAX, where = 0;  // rows that are not there need no mask: nothing of theirs is kept
      float mul = 1.f, rowf = 0.f, slope = 0.f;
      int64_t out_row = 0;
      const bool special = (p.softcap > 0.f || p.slopes != nullptr) && __any_sync(0xffffffffu, there);
      const float cap = p.softcap * kLog2e;
      uint8_t* my_q = smem + tile * C::kQ + (r & 127) * 16;
      if (there) {
        const int i = p.cu_q ? rr / p.group : 0, head = h * p.group + (rr - i * p.group);
        const QuerySpan s = query_span(p, b, i, q);
        lo = s.lo, hi = s.hi, where = s.pos;
        out_row = (q.q0 + i) * p.q_heads + head;
        slope = p.slopes ? p.slopes[head] * kLog2e : 0.f;
        const int64_t src = (q.q0 + i) * p.q_st + (int64_t)head * p.q_sh;
        // the row's 16-byte pieces, all in flight at once (heads of 256: in two halves, the second time from cache)
        constexpr int kPieces = D / 8, kOnce = kPieces > 16 ? 16 : kPieces;
        uint4 raw[kOnce];
        auto load = [&](int c0) {
          const uint4* at = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + src) + c0;
#pragma unroll
          for (int c = 0; c < kOnce; ++c) raw[c] = __ldg(at + c);
        };
        // values 2i, 2i + 1 of the pieces held
        auto pair = [&](int i) -> float2 {
          const uint4 x = raw[i / 4];
          const uint32_t w = (i & 3) == 0 ? x.x : (i & 3) == 1 ? x.y : (i & 3) == 2 ? x.z : x.w;
          if (p.dtype == B2Q_DTYPE_F16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
          return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
        };
        float top = 0.f;
#pragma unroll
        for (int c0 = kPieces - kOnce; c0 >= 0; c0 -= kOnce) {
          load(c0);
#pragma unroll
          for (int i = 0; i < kOnce * 4; ++i) {
            const float2 v = pair(i);
            top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
          }
        }
        // to 2^6 .. 2^7: products with keys of up to 2^16 stay far below f32's range
        const int e2 = max(-100, (__float_as_int(top) >> 23) - 127);
        const float up = __int_as_float((127 + 6 - e2) << 23);
        rowf = __int_as_float((127 + e2 - 6) << 23) * p.scale;
        rowf *= p.softcap > 0.f ? 1.f / p.softcap : kLog2e;
        rowf = fminf(rowf, FLT_MAX);  // (times a score of 0)
        mul = rowf;
#pragma unroll
        for (int c0 = 0; c0 < kPieces; c0 += kOnce) {
          if (c0 > 0) load(c0);
#pragma unroll
          for (int w = 0; w < kOnce; ++w) {  // chunk (t, block) = a word of a packed key: its 8 values in its order
            const int k = w / 4, t = w & 3;
            // first and second run of 4 values
            float2 a0 = pair(16 * k + (FMT == 0 ? 2 : 4) * t), a1 = pair(16 * k + (FMT == 0 ? 2 : 4) * t + 1);
            float2 z0 = pair(16 * k + (FMT == 0 ? 8 + 2 * t : 4 * t + 2)), z1 = pair(16 * k + (FMT == 0 ? 9 + 2 * t : 4 * t + 3));
            a0.x *= up, a0.y *= up, a1.x *= up, a1.y *= up, z0.x *= up, z0.y *= up, z1.x *= up, z1.y *= up;
            uint4 x;
            if (FMT == 0)
              x = make_uint4(pack_half2(a0.x, a1.x), pack_half2(z0.x, z1.x), pack_half2(a0.y, a1.y), pack_half2(z0.y, z1.y));
            else
              x = make_uint4(pack_half2(a0.x, a0.y), pack_half2(a1.x, a1.y), pack_half2(z0.x, z0.y), pack_half2(z1.x, z1.y));
            *reinterpret_cast<uint4*>(my_q + (t * NB + c0 / 4 + k) * 2048) = x;
          }
        }
      } else if (tile < tiles) {
#pragma unroll 2
        for (int w = 0; w < NB * 4; ++w) *reinterpret_cast<uint4*>(my_q + w * 2048) = make_uint4(0, 0, 0, 0);
      }
      __syncwarp();
      tc::fence_async_smem();
      tc::arrive(smem_addr(&b_q));
      if (tile < tiles) {
        // the weights of 32 keys: 16 registers of pairs, and (WIDE) 16 more of what their rounding left
        constexpr int kWords = WIDE ? 32 : 16;
        auto put = [](uint32_t (&w)[kWords], int i, float y0, float y1) {
          w[i] = pack_half2(y0, y1);
          if constexpr (WIDE) {
            const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            w[16 + i] = pack_half2(y0 - back.x, y1 - back.y);
          }
        };
        auto store = [&](int c, const uint32_t (&w)[kWords]) {
          if constexpr (WIDE)
            tc::tmem_st32(col_s + c, w);
          else
            tc::tmem_st16(col_s + c / 2, w);
        };
        float ref = kNoRef, sum = 0.f;
        for (int j = 0; j < n; ++j) {
          if (!wait(&b_s[tile], done_blocks[tile] + j)) break;
          tc::fence_after();
          const int kb = (begin + j) * STG;
          const int turn = (blocks + j) & 3;
          const uint4 odds = *reinterpret_cast<const uint4*>(s_odd[turn]);
          const bool odd = (odds.x | odds.y | odds.z | odds.w) != 0;
          // masked or special scores are finished in the first pass and put back
          const bool mask = __any_sync(0xffffffffu, kb < lo || kb + STG > hi);
          const bool careful = special || mask;
          const float scale = careful ? 1.f : mul;
          // takes the reference to 2^-7 of the row's maximum where that has grown by more than 2^8, and O with it: a row's
          // largest weight lies from 2^7 to 2^15, and weights down to 2^-21 of it keep all of f16's bits
          auto follow = [&](float top) {
            const bool grown = top > ref + 15.f;
            if (!__any_sync(0xffffffffu, grown)) return;
            const float now = grown ? top - 7.f : ref, f = exp2_approx(ref - now);
            ref = now, sum *= f;
            if (j > 0) {  // the block before is in O already: its product ended before this block's scores
#pragma unroll 1
              for (int c = 0; c < D; c += 32) {
                uint32_t v[32];
                tc::tmem_ld32_nowait(col_o + c, v);
                tc::tmem_wait_ld32(v);
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
                tc::tmem_st32(col_o + c, v);
              }
            }
          };
          if (__builtin_expect(odd, 0)) {  // the two passes below, an element at a time
            float top = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < STG; c += 32) {
              const uint32_t odds = s_odd[turn][c >> 5], large_k = odds ? s_less[turn][0][c >> 5] : 0,
                             large_v = odds ? s_less[turn][1][c >> 5] : 0, unread = odds & ~(large_k | large_v);
              uint32_t x[32];
              tc::tmem_ld32_nowait(col_s + c, x);
              tc::tmem_wait_ld32(x);
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                float y = __uint_as_float(x[e]) * (large_k >> e & 1 ? rowf * (float)(1 << C::kLess) : rowf);
                if (p.softcap > 0.f) y = cap * (fabsf(y) <= kTanhLimit ? tanh_near(y) : tanh_far(y));
                if (p.slopes) y = fmaf(-slope, fabsf((float)(where - kb - c - e)), y);
                if (kb + c + e < lo || kb + c + e >= hi || (unread >> e & 1)) y = -INFINITY;
                top = fmaxf(top, large_v >> e & 1 ? y + C::kLess : y);
                x[e] = __float_as_uint(y);
              }
              tc::tmem_st32(col_s + c, x);
            }
            tc::tmem_wait_st();
            follow(top);
#pragma unroll 1
            for (int c = 0; c < STG; c += 32) {
              const uint32_t large_v = s_odd[turn][c >> 5] ? s_less[turn][1][c >> 5] : 0;
              uint32_t x[32], w[kWords];
              tc::tmem_ld32_nowait(col_s + c, x);
              tc::tmem_wait_ld32(x);
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float y0 = exp2_approx(__uint_as_float(x[e]) - ref), y1 = exp2_approx(__uint_as_float(x[e + 1]) - ref);
                sum += y0 + y1;
                put(w, e / 2, large_v >> e & 1 ? y0 * (float)(1 << C::kLess) : y0,
                    large_v >> (e + 1) & 1 ? y1 * (float)(1 << C::kLess) : y1);
              }
              store(c, w);
            }
            tc::tmem_wait_st();
            tc::fence_before();
            tc::arrive(smem_addr(&b_p[tile]));
            continue;
          }
          // Two passes over S, 32 columns at a time: for the maximum (masked and special scores are finished then, and put
          // back), and for the weights.
          float top = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < STG; c += 32) {
            uint32_t x[32];
            tc::tmem_ld32_nowait(col_s + c, x);
            tc::tmem_wait_ld32(x);
            if (careful) {
              const float2 rowf2 = make_float2(rowf, rowf);
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float2 y = __fmul2_rn(make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), rowf2);
                x[e] = __float_as_uint(y.x), x[e + 1] = __float_as_uint(y.y);
              }
              if (p.softcap > 0.f) {  // rowf made these the cap's arguments
                float far = 0.f;
#pragma unroll
                for (int e = 0; e < 32; ++e) far = fmaxf(far, fabsf(__uint_as_float(x[e])));
                if (!__any_sync(0xffffffffu, far > kTanhLimit)) {
#pragma unroll
                  for (int e = 0; e < 32; e += 2) {  // cap * tanh_near, two at a time
                    const float2 z = make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), u = __fmul2_rn(z, z);
                    float2 y = make_float2(kTanh4, kTanh4);
                    y = __ffma2_rn(y, u, make_float2(kTanh3, kTanh3));
                    y = __ffma2_rn(y, u, make_float2(kTanh2, kTanh2));
                    y = __ffma2_rn(y, u, make_float2(kTanh1, kTanh1));
                    y = __ffma2_rn(y, u, make_float2(kTanh0, kTanh0));
                    y = __fmul2_rn(y, __fmul2_rn(z, make_float2(cap, cap)));
                    x[e] = __float_as_uint(y.x), x[e + 1] = __float_as_uint(y.y);
                  }
                } else {
#pragma unroll
                  for (int e = 0; e < 32; ++e) {
                    const float z = __uint_as_float(x[e]);
                    x[e] = __float_as_uint(cap * (fabsf(z) <= kTanhLimit ? tanh_near(z) : tanh_far(z)));
                  }
                }
              }
              if (p.slopes) {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  x[e] = __float_as_uint(fmaf(-slope, fabsf((float)(where - kb - c - e)), __uint_as_float(x[e])));
              }
              if (mask) {
                const int from_e = lo - kb - c, to_e = hi - kb - c;
#pragma unroll
                for (int e = 0; e < 32; ++e) x[e] = e >= from_e && e < to_e ? x[e] : 0xff800000u;
              }
              tc::tmem_st32(col_s + c, x);
            }
#pragma unroll
            for (int e = 0; e < 32; e += 2) top = fmaxf(top, fmaxf(__uint_as_float(x[e]), __uint_as_float(x[e + 1])));
          }
          if (careful) tc::tmem_wait_st();
          follow(top * scale);
          float2 s01 = make_float2(0.f, 0.f);
          const float2 scale2 = make_float2(scale, scale), ref2 = make_float2(-ref, -ref);
#pragma unroll 1
          for (int c = 0; c < STG; c += 32) {
            uint32_t x[32], w[kWords];
            tc::tmem_ld32_nowait(col_s + c, x);
            tc::tmem_wait_ld32(x);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float2 y = make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1]));
              y = __ffma2_rn(y, scale2, ref2);
              y.x = exp2_approx(y.x), y.y = exp2_approx(y.y);
              s01 = __fadd2_rn(s01, y);
              put(w, e / 2, y.x, y.y);
            }
            store(c, w);  // to columns of S that have been read
          }
          sum += s01.x + s01.y;
          tc::tmem_wait_st();
          tc::fence_before();
          tc::arrive(smem_addr(&b_p[tile]));
        }
        // ---------------------------------------------------------- the row's result, or this share's part of it
        if (wait(&b_o[tile], done_tiles[tile])) {
          tc::fence_after();
          const bool begun = from > 0, done = to == span.count;
          const int part = 2 * (int)blockIdx.x + (begun ? 0 : 1);
          const bool final = !begun && done;
          const float inv = !final ? 1.f : (sum > 0.f || sum != sum ? __fdividef(1.f, sum) : 0.f);
          float* dst = p.part_o + ((int64_t)part * R + r) * D;
#pragma unroll 1
          for (int k = 0; k < NB; ++k) {
            uint32_t v[32];
            tc::tmem_ld32_nowait(col_o + k * 32, v);
            tc::tmem_wait_ld32(v);
            if (there) {
              // columns of a block: q4_0 [nibble][g] of values 2g, 16+2g, 2g+1, 17+2g; q8_0 [i][g] of values 4g + i
              float y[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const int g = e & 7, i = e >> 3;
                y[FMT == 0 ? 2 * g + (i >> 1) + 16 * (i & 1) : 4 * g + i] = __uint_as_float(v[e]) * inv;
              }
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                if (!final)
                  store4(dst + k * 32 + e, y[e], y[e + 1], y[e + 2], y[e + 3]);
                else if (p.dtype == B2Q_DTYPE_F16)
                  store4(static_cast<__half*>(p.out) + out_row * D + k * 32 + e, y[e], y[e + 1], y[e + 2], y[e + 3]);
                else
                  store4(static_cast<__nv_bfloat16*>(p.out) + out_row * D + k * 32 + e, y[e], y[e + 1], y[e + 2],
                         y[e + 3]);
              }
            }
          }
          if (there && !final) p.part_m[part * R + r] = make_float2(ref, sum);
          if (there && final && p.lse) p.lse[out_row] = (ref + log2f(sum)) * kLn2;
          tc::fence_before();
        }
      }
    } else if constexpr (ROLE == 1) {
      // ------------------------------------------------------------ unpacking: a thread a key, then 8 keys' columns
      const int th = threadIdx.x - SW * 32, kg = th >> 3, g = th & 7;
      const int32_t* table = p.table + (int64_t)b * p.table_stride;
      constexpr int UV = FMT == 0 ? NB * 2 : NB * 4;  // bytes of a value unit's slice of a row
      // the row (of heads' tokens) of a token of this KV head, or -1
      auto row_of = [&](int tok) -> int64_t {
        if (tok >= q.len) return -1;
        const int id = table[tok >> p.page_shift];
        if (id < 0 || id >= p.pages) {
          atomicCAS(&g_device_error, 0, kErrPage);
          return -1;
        }
        return ((((int64_t)id * p.heads) + h) << p.page_shift) + (tok & ((1 << p.page_shift) - 1));
      };
      uint32_t kw[C::kRow / 4], ksc[(NB + 1) / 2], kvs[(NB + 1) / 2];  // a key's row, its scales, its value's scales
      uint32_t vw[8][(UV + 3) / 4], vsc[8][(NB + 1) / 2];
      bool read_k = false;
      int read_v = 0;  // of the 8 keys
      auto load_k = [&](int j) {
        const int64_t row = j < n ? row_of((begin + j) * STG + th) : -1;
        read_k = row >= 0;
        if (read_k) {
          ldg_bytes<C::kRow>(p.kq + row * C::kRow, kw);
          ldg_bytes<NB * 2>(reinterpret_cast<const uint8_t*>(p.ks + row * NB), ksc);
          ldg_bytes<NB * 2>(reinterpret_cast<const uint8_t*>(p.vs + row * NB), kvs);
        } else {  // zeros, whatever the quants held are
#pragma unroll
          for (int k = 0; k < (NB + 1) / 2; ++k) ksc[k] = kvs[k] = 0;
        }
      };
      auto load_v = [&](int j) {
        const int tok = (begin + j) * STG + kg * 8;
        const int64_t row = j < n ? row_of(tok) : -1;
        read_v = row >= 0 ? min(8, q.len - tok) : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < read_v) {
            ldg_bytes<UV>(p.vq + (row + i) * C::kRow + g * UV, vw[i]);
            ldg_bytes<NB * 2>(reinterpret_cast<const uint8_t*>(p.vs + (row + i) * NB), vsc[i]);
          } else {
#pragma unroll
            for (int k = 0; k < (NB + 1) / 2; ++k) vsc[i][k] = 0;
          }
      };
      constexpr uint32_t kOne = 0x3c003c00u, kLessHalf = (15 - C::kLess) << 10;  // f16: 1 and 1, 2^-kLess
      load_k(0);
      if (FMT == 0) load_v(0);  // q8_0: no registers to have them a block ahead
      for (int j = 0; j < n && ok; ++j) {
        const uint32_t at = blocks + j;
        const int vbuf = at % VB;
        if (FMT == 2) load_v(j);
        const uint32_t largest_k = largest_half<NB>(ksc), largest_v = largest_half<NB>(kvs);
        const bool large = max(largest_k, largest_v) > C::kMost;  // or not finite
        const uint32_t odd = __ballot_sync(0xffffffffu, large || (!read_k && (begin + j) * STG + th < q.len));
        bool gone = false;
#pragma unroll 1
        for (int turn = 0; turn < TURNS; ++turn) {
          const uint32_t use = at * TURNS + turn;  // of the key tiles
          const int kbuf = use % KB;
          if (use >= KB && !wait(&b_kempty[kbuf], use / KB - 1)) {
            gone = true;
            break;
          }
          if (lane == 0) s_odd[at & 3][warp - SW] = odd;
          uint8_t* kt = smem + MT * C::kQ + kbuf * (C::kParts / TURNS) * C::kTile + th * 16;
          // word w = (t, block) of the key, its packed quants and its scale -> the operand's 16 bytes
          auto unpack_key = [&](int w, uint32_t q0, uint32_t q1, uint32_t d, uint32_t less) {
            uint32_t i[4], x[4];  // the quants as f16, and times their scale
            if constexpr (FMT == 0) {
              i[0] = low_nibbles<true>(q0), i[1] = high_nibbles_int(q0);
              i[2] = low_nibbles<true>(q0 >> 8), i[3] = high_nibbles_int(q0 >> 8);
            } else {
              i[0] = two_bytes<true>(q0, 0), i[1] = two_bytes<true>(q0, 1);
              i[2] = two_bytes<true>(q1, 0), i[3] = two_bytes<true>(q1, 1);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (less != kOne) i[e] = mul_half2(i[e], less);
              x[e] = mul_half2(i[e], d);
            }
            if (TURNS == 1 || turn == 0) *reinterpret_cast<uint4*>(kt + w * 2048) = make_uint4(x[0], x[1], x[2], x[3]);
            if (EXACT && (TURNS == 1 || turn == 1)) {  // what the rounding left: one exact fused multiply-add
#pragma unroll
              for (int e = 0; e < 4; ++e) x[e] = fma_half2(i[e], d, x[e] ^ 0x80008000u);
              *reinterpret_cast<uint4*>(kt + (TURNS == 1 ? C::kTile : 0) + w * 2048) = make_uint4(x[0], x[1], x[2], x[3]);
            }
          };
#pragma unroll
          for (int w = 0; w < NB * 4; ++w) {
            const int k = w % NB;
            unpack_key(w, kw[FMT == 0 ? w : 2 * w], FMT == 0 ? 0 : kw[2 * w + 1],
                       __byte_perm(ksc[k / 2], 0, (k & 1) ? 0x3232 : 0x1010), kOne);
          }
          if (__builtin_expect(odd != 0, 0)) {
            const uint32_t k = __ballot_sync(0xffffffffu, largest_k > C::kMost), v = __ballot_sync(0xffffffffu, largest_v > C::kMost);
            if (lane == 0) s_less[at & 3][0][warp - SW] = k, s_less[at & 3][1][warp - SW] = v;
            if (large) {  // once more: 2^kLess less, or NaN where a scale is not finite, and so the rows that see this key
              const int64_t row = row_of((begin + j) * STG + th);
              const bool finite = max(largest_k, largest_v) < 0x7c00u;
              const uint32_t less = largest_k > C::kMost ? kLessHalf * 0x10001u : kOne;
#pragma unroll 1
              for (int w = 0; w < NB * 4; ++w) {
                const uint8_t* at = p.kq + row * C::kRow + w * (C::kRow / (NB * 4));
                const uint32_t q0 = __ldg(reinterpret_cast<const uint32_t*>(at));
                const uint32_t q1 = FMT == 0 ? 0 : __ldg(reinterpret_cast<const uint32_t*>(at) + 1);
                unpack_key(w, q0, q1, finite ? p.ks[row * NB + w % NB] * 0x10001u : 0x7fff7fffu, less);
              }
            }
          }
          if (turn + 1 == TURNS) load_k(j + 1);
          tc::fence_async_smem();
          tc::arrive(smem_addr(&b_kfull[kbuf]));
        }
        if (gone) break;

        if (at >= VB && !wait(&b_vempty[vbuf], at / VB - 1)) break;
        uint8_t* vt = smem + MT * C::kQ + (C::kHeld + vbuf) * C::kTile + kg * (D * 16) + g * 16;
        // column 4k + c of the unit: 8 keys' values, from two keys' packed quants and scales at a time
        auto unpack_values = [&](uint32_t w0, uint32_t w1, int odd_block, uint32_t d, uint32_t less, uint32_t (&x)[4]) {
          if constexpr (FMT == 0) {
            const uint32_t w = __byte_perm(w0, w1, odd_block ? 0x7632 : 0x5410);
            x[0] = low_nibbles<true>(w), x[1] = high_nibbles_int(w);
            x[2] = low_nibbles<true>(w >> 8), x[3] = high_nibbles_int(w >> 8);
          } else {
            const uint32_t lo = __byte_perm(w0, w1, 0x5140), hi = __byte_perm(w0, w1, 0x7362);
            x[0] = two_bytes<true>(lo, 0), x[1] = two_bytes<true>(lo, 1);
            x[2] = two_bytes<true>(hi, 0), x[3] = two_bytes<true>(hi, 1);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) x[c] = mul_half2(less != kOne ? mul_half2(x[c], less) : x[c], d);
        };
        auto store_values = [&](int k, const uint32_t (&x)[4][4]) {  // [pair of keys][column]
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint4*>(vt + (k * 32 + c * 8) * 16) = make_uint4(x[0][c], x[1][c], x[2][c], x[3][c]);
        };
        uint32_t top = vsc[0][0] & 0x7fff7fffu;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int k = 0; k < (NB + 1) / 2; ++k) top = __vmaxu2(top, vsc[i][k] & 0x7fff7fffu);
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          uint32_t x[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int word = FMT == 0 ? k / 2 : k;
            unpack_values(vw[2 * i][word], vw[2 * i + 1][word], k & 1,
                          __byte_perm(vsc[2 * i][k / 2], vsc[2 * i + 1][k / 2], (k & 1) ? 0x7632 : 0x5410), kOne, x[i]);
          }
          store_values(k, x);
        }
        if (__builtin_expect(max(top & 0xffffu, top >> 16) > C::kMost, 0)) {
          // once more: rows with a large scale 2^kLess less, those with one that is not finite zeros (their keys are NaN)
          const int64_t row = row_of((begin + j) * STG + kg * 8);
          uint32_t use = 0, large = 0;
#pragma unroll 1
          for (int i = 0; i < read_v; ++i) {
            uint32_t m = 0;
#pragma unroll 1
            for (int k = 0; k < NB; ++k) m = max(m, p.vs[(row + i) * NB + k] & 0x7fffu);
            use |= (m < 0x7c00u) << i, large |= (m > C::kMost) << i;
          }
#pragma unroll 1
          for (int k = 0; k < NB; ++k) {
            uint32_t x[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t w[2], d[2], less[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int key = 2 * i + e;
                const bool is = use >> key & 1;
                const uint8_t* at = p.vq + (row + (is ? key : 0)) * C::kRow + g * UV + k * (UV / NB);
                w[e] = FMT == 0 ? *reinterpret_cast<const uint16_t*>(at) : *reinterpret_cast<const uint32_t*>(at);
                d[e] = is ? p.vs[(row + key) * NB + k] : 0;
                less[e] = large >> key & 1 ? kLessHalf : 0x3c00u;
              }
              unpack_values(w[0], w[1], 0, d[0] | d[1] << 16, less[0] | less[1] << 16, x[i]);
            }
            store_values(k, x);
          }
        }
        if (FMT == 0) load_v(j + 1);
        tc::fence_async_smem();
        tc::arrive(smem_addr(&b_vfull[vbuf]));
      }
    } else if (warp == SW + 4 && lane == 0) {
      // ------------------------------------------------------------ the products, issued in the order in which they run
      const uint32_t is = tc::instr_desc_f16(STG), io = tc::instr_desc_f16(D);
      const uint64_t dq = tc::smem_desc_kmajor(q_smem, 2048), dk = tc::smem_desc_kmajor(k_smem, 2048);
      const uint64_t dv = tc::smem_desc_kmajor(v_smem, D * 16);
      auto scores = [&](int tile, uint32_t at) {
        const uint64_t a = dq + (uint64_t)((tile * C::kQ) >> 4);
        const uint64_t z = dk + (uint64_t)((at * TURNS % KB * (C::kParts / TURNS) * C::kTile) >> 4);
#pragma unroll
        for (int part = 0; part < C::kParts; ++part) {
          if (TURNS == 2 && part == 1) {  // its turn comes when the first part has been read
            tc::mma_commit(smem_addr(&b_kempty[0]));
            if (!wait_one(&b_kfull[0], at * TURNS + 1)) return;
            tc::fence_after();
          }
#pragma unroll
          for (int s = 0; s < D / 16; ++s)
            tc::mma_f16_ss(tmem + C::kS + tile * 128, a + s * (4096 >> 4),
                           z + (((TURNS == 1 ? part * C::kTile : 0) + s * 4096) >> 4), is, part > 0 || s > 0);
        }
        tc::mma_commit(smem_addr(&b_s[tile]));
        tc::arrive(smem_addr(&b_s[tile]));
      };
      if (wait_one(&b_q, segments) && wait_one(&b_kfull[blocks * TURNS % KB], blocks * TURNS / KB)) {
        tc::fence_after();
        for (int i = 0; i < tiles; ++i) scores(i, blocks);
        tc::mma_commit(smem_addr(&b_kempty[blocks * TURNS % KB]));
        for (int j = 0; j < n && ok; ++j) {
          const uint32_t at = blocks + j;
          for (int i = 0; i < tiles; ++i) {
            if (i == 0 && !wait_one(&b_vfull[at % VB], at / VB)) break;
            if (!wait_one(&b_p[i], done_blocks[i] + j)) break;
            tc::fence_after();
            const uint64_t z = dv + (uint64_t)(((at % VB) * C::kTile) >> 4);
#pragma unroll
            for (int s = 0; s < STG / 16; ++s)
              if constexpr (WIDE) {
#pragma unroll
                for (int part = 0; part < 2; ++part)
                  tc::mma_f16_ts(tmem + i * 128, tmem + C::kS + i * 128 + s / 2 * 32 + part * 16 + s % 2 * 8,
                                 z + (uint64_t)s * ((2 * D * 16) >> 4), io, j > 0 || s > 0 || part > 0);
              } else {
                tc::mma_f16_ts(tmem + i * 128, tmem + C::kS + i * 128 + s * 8, z + (uint64_t)s * ((2 * D * 16) >> 4), io,
                               j > 0 || s > 0);
              }
            if (j + 1 == n) {
              tc::mma_commit(smem_addr(&b_o[i]));
            } else {
              if (i == 0 && !wait_one(&b_kfull[(at + 1) * TURNS % KB], (at + 1) * TURNS / KB)) break;
              tc::fence_after();
              scores(i, at + 1);
            }
          }
          if (!ok) break;
          tc::mma_commit(smem_addr(&b_vempty[at % VB]));
          if (j + 1 < n) tc::mma_commit(smem_addr(&b_kempty[(at + 1) * TURNS % KB]));
        }
      }
    }

    const bool begun = from > 0, done = to == span.count;
    if (begun && done && threadIdx.x == 0) {  // this CTA ends a tile that others began: the joining kernel's work
      join.first = (int)((pos - skip + p.tile_cost) / share.per);
      join.rows = min(rows, R), join.row0 = rt * R, join.head0 = h * p.group, join.q0 = (int)q.q0;
    }
    blocks += n, ++segments;
    for (int i = 0; i < tiles; ++i) done_blocks[i] += n, ++done_tiles[i];
    pos += take, skip += take;
    if (skip == units) skip = 0, ++h;
    tc::fence_before();
    __syncwarp();
    asm volatile("bar.sync 1, %0;" ::"n"(C::kWarps * 32) : "memory");  // the queries' memory, O and S are free
    tc::fence_after();
    if (s_abort) break;
  }
  if (ROLE == 0 && threadIdx.x == 0) {
    if (s_abort) join.first = -1;
    p.joins[blockIdx.x] = join;
  }
  };
  if (warp < SW) {
    if constexpr (MT == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
    work(std::integral_constant<int, 0>{});
  } else if (warp < SW + 4) {
    work(std::integral_constant<int, 1>{});
  } else {
    if constexpr (MT == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kIssueRegs));
    work(std::integral_constant<int, 2>{});
  }
  // nothing is in flight: a segment ends when its last products have been waited for. Where a wait ran out, they may not
  // have: let the products issued so far end (they need nothing more) before their memory goes away.
  if (s_abort) {
    if (warp == SW + 4 && lane == 0) {
      tc::mma_commit(smem_addr(&b_end));
      mbar_wait(smem_addr(&b_end), 0, kWaitLimit);
    }
    if (threadIdx.x == 0) atomicCAS(&g_device_error, 0, kErrTimeout);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

template <int FMT, int NB, bool EXACT, bool WIDE>
static int launch_attention_tc_as(const AttnParams& p, int sms, cudaStream_t stream) {
  using C = TcTile<FMT, NB, EXACT>;
  static_assert(C::kSmem + 2048 <= 227 * 1024, "shared memory of a CTA");
  auto kernel = attention_tc_kernel<FMT, NB, EXACT, WIDE>;
  static std::atomic<unsigned long long> allowed{0};
  int rc = allow_smem_once(reinterpret_cast<const void*>(kernel), C::kSmem, allowed);
  if (rc) return rc;
  if (C::MT == 2) {  // the split waits for registers that the block was not launched with: never launch it short of them
    static std::atomic<int> regs{0};
    if (!regs.load(std::memory_order_relaxed)) {
      cudaFuncAttributes attr;
      const cudaError_t e = cudaFuncGetAttributes(&attr, kernel);
      if (e != cudaSuccess) return fail(B2Q_ECUDA, "b2q_attention: %s", cudaGetErrorString(e));
      regs.store(attr.numRegs, std::memory_order_relaxed);
    }
    if (regs.load(std::memory_order_relaxed) != C::kLaunchRegs)
      return fail(B2Q_ECUDA, "b2q_attention: built with %d registers a thread, not %d",
                  regs.load(std::memory_order_relaxed), C::kLaunchRegs);
  }
  launch_maybe_pdl(kernel, dim3((unsigned)sms), dim3(C::kWarps * 32), C::kSmem, stream, p);
  rc = after_launch("attention_tc");
  if (rc) return rc;
  launch_maybe_pdl(attention_join_kernel<NB, C::kRows>, dim3((unsigned)sms, 16), dim3(128), 0, stream, p);
  return after_launch("attention_join");
}

template <int FMT>
static int launch_attention_tc_fmt(AttnParams p, int dim, int sms, cudaStream_t stream) {
  p.tile_cost = tc_tile_cost(p);
  const bool wide = p.dtype == B2Q_DTYPE_F16, exact = wide || p.lse;
  auto by_parts = [&](auto nb) {
    constexpr int NB = decltype(nb)::value;
    if constexpr (NB == 8)
      return wide ? launch_attention_tc_as<FMT, NB, true, true>(p, sms, stream) : launch_attention_tc_as<FMT, NB, false, false>(p, sms, stream);
    else
      return wide    ? launch_attention_tc_as<FMT, NB, true, true>(p, sms, stream)
             : exact ? launch_attention_tc_as<FMT, NB, true, false>(p, sms, stream)
                     : launch_attention_tc_as<FMT, NB, false, false>(p, sms, stream);
  };
  switch (dim) {
    case 64: return by_parts(std::integral_constant<int, 2>{});
    case 96: return by_parts(std::integral_constant<int, 3>{});
    case 128: return by_parts(std::integral_constant<int, 4>{});
    default: return by_parts(std::integral_constant<int, 8>{});
  }
}

}  // namespace b2q
