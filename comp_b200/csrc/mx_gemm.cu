// Products of MXFP4 operands on the fifth-generation tensor cores, for one weight matrix or for an expert's each.
//
//   y[r][n] = sum over blocks of 2^(sx - 127) 2^(sw - 127) * sum over the block of x w
//
// tcgen05.mma kind::mxf4 multiplies 128 weight rows by up to 256 rows of x, 64 values of K at a time, applies both operands'
// block scales and adds in f32: no thread touches an operand. Weights are the operand with 128 rows even for a single row of
// x, since the unit's other side may be as few as 16 rows, and each lane of tensor memory then is a column n of y, so that a
// warp's stores of a row of y are runs of 32 values.
//
// A tile is 128 weight rows by TN rows of x of one expert; CTAs are persistent and take tiles in turn. Three roles:
//   - one thread copies stages (256 values of K: codes and scales as they lie in the operand images) into a ring of shared
//     memory, one bulk copy an operand and 128 rows;
//   - one thread copies a stage's scales on into tensor memory and issues its four products;
//   - four warps turn the previous tile's accumulator into rows of y, while the next tile's products run. An accumulator of
//     256 columns and a second one do not fit beside the scales (512 columns in all): the second begins 64 columns before the
//     first one's end, and those are read first.
// Few tiles (narrow layers, few rows) leave most of the GPU idle: then the CTAs of a cluster split K between them, and add
// their parts in order of rank through distributed shared memory, so that results do not depend on timing.
// (They hold tensor memory while they wait for one another, which is safe only because none of them ever waits for any: beside
// its 205 KB of shared memory and more an SM has no room for another kernel that takes tensor memory, whose least is 28.)
//
// What bounds it: a stage of 256 rows writes 51 KB into shared memory and the products read 49 KB of it, 790 cycles at 128 bytes a
// cycle, where the products alone would take 512; measured 745 to 820, at 1.6 to 1.7 GHz under the power limit: 4096 x 14336 x
// 4096 103 us (4.7 PFLOP/s), 118 in a long run; 8192 x 8192 x 8192 209 us (5.3). With few rows the weights' stream: 64 tokens of 8
// among 128 experts of 4096 x 2048 97 us (5.8 TB/s). In between the steps that follow one another: 8192 x 8192 with 16 / 64 / 256 rows
// 11.7 / 13.8 / 17.9 us, where the weights take 5.5: the quantizer's launch 2.5, 128 of 148 SMs at work (64 row tiles, K or
// the rows of x in two), the join of the parts of K 1 + n / 50.
#include <algorithm>
#include <atomic>

#include "mx_tiles.cuh"

namespace b2q {

namespace {

// TN is 64 at least: a tile's rows may begin inside the 128 whose scales lie in four columns of tensor memory, and the
// products take scales from even columns only, which is every 64 rows.
template <int TN>
struct MxTile {
  static_assert(TN == 64 || TN == 128 || TN == 256, "rows of a tile");
  static constexpr int kParts = (TN + 127) / 128;             // x tiles of 128 rows
  static constexpr int kXCodes = TN * 128;                    // bytes of a stage: codes and scales of x
  static constexpr int kStageBytes = kMxBytes + kXCodes + kParts * 1024;
  static constexpr int kStages = TN == 64 ? 8 : TN == 128 ? 6 : 4;
  static constexpr int kSmem = kStages * kStageBytes + 1024;  // 1024: the ring begins at a multiple of that
  static constexpr uint32_t kSecond = TN == 256 ? 192 : TN;   // column of the second accumulator
  static constexpr uint32_t kScaleCol = 448;                  // scales: two sets, which stages take in turn
  static constexpr uint32_t kScaleSet = 8 + kParts * 8;
  static_assert(kSecond + TN <= kScaleCol && kScaleCol + 2 * kScaleSet <= 512, "tensor memory");
  static_assert(kSmem <= 227 * 1024 - 13 * 1024, "shared memory");  // beside it: the experts' table
  static_assert(kSmem >= 200 * 1024, "one CTA with tensor memory an SM");  // of 228 KB: the others' take 28 at the least
};

constexpr int kThreads = 192;

__device__ __forceinline__ void arrive_bar(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 32 consecutive columns of this thread's lane
__device__ __forceinline__ void load_columns(uint32_t taddr, uint32_t (&a)[16], uint32_t (&b)[16]) {
  tc::tmem_ld16_nowait(taddr, a);
  tc::tmem_ld16_nowait(taddr + 16, b);
  tc::tmem_wait_ld_regs(a);
  tc::regs_ready(b);
}

template <int TN, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) mx_gemm_kernel(const MxGemm g) {
  using C = MxTile<TN>;
  constexpr int S = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t b_full[S], b_empty[S], b_acc[2], b_free[2], b_end;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_tiles, s_warp[kThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = (smem_addr(smem_raw) + 1023) & ~1023u;
  int* table = reinterpret_cast<int*>(smem_raw + C::kSmem);
  uint32_t rank = 0, ranks = 1;
  if (SPLIT) {
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  }

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s_tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) mbar_init(smem_addr(&b_full[i]), 1), mbar_init(smem_addr(&b_empty[i]), 1);
    for (int i = 0; i < 2; ++i) mbar_init(smem_addr(&b_acc[i]), 1), mbar_init(smem_addr(&b_free[i]), 128);
    mbar_init(smem_addr(&b_end), 1);
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (!g.early) asm volatile("griddepcontrol.wait;" ::: "memory");
  const int units = g.row_tiles;
  const Experts experts = count_tiles<TN, kThreads>(g, table, s_warp, &s_tiles, units);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = s_tmem;
  const int tiles = s_tiles, step = gridDim.x / ranks, start = blockIdx.x / ranks;
  const int k0 = (int)((int64_t)g.stages * rank / ranks), k1 = (int)((int64_t)g.stages * (rank + 1) / ranks);
  // The next kernel may start only once this CTA has its tensor memory: one that took tensor memory first and then waited
  // for this grid would leave both waiting.
  if (warp != 0) asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  bool ok = true;
  // a wait that ran out ends the role's work: every later one is skipped
  auto wait_warp = [&](uint64_t* bar, uint32_t phase) {
    if (ok) {
      ok = __all_sync(0xffffffffu, mbar_wait(smem_addr(bar), phase & 1, kWaitLimit));
      if (!ok) atomicExch(&s_abort, 1);
    }
    return ok;
  };

  uint32_t it = 0, tile_count = 0;  // stages and tiles so far: the barriers' phases
  bool waited = !g.early;
  for (int t = start; t < tiles; t += step) {
    const TileAt at = tile_at<TN>(g, experts, t, units);
    if (warp == 0) {
      // rows of x, and weights that several tiles read, are to stay in L2 (4096 x 14336 x 4096 115 -> 112 us with the quantizer)
      const uint64_t once = evict_first_policy();
      uint64_t keep;
      asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(keep));
      const uint64_t w_policy = at.again ? keep : once;
      const int parts = (at.n + 127) >> 7;
      // of the rows' codes no more than the products read (which is up to 8 rows more, left from other stages)
      const uint32_t codes = (uint32_t)((at.n + 7) & ~7) * 128, bytes = kMxBytes + codes + parts * 1024;
      const uint8_t* w = g.w + ((int64_t)at.e * units + at.rt) * g.stages * kMxBytes;
      const uint8_t* x = g.x + (int64_t)at.x_tile * g.stages * kMxBytes;
      auto copy_x = [&](uint32_t stage, uint32_t bar, int k) {
        const uint8_t* src = x + (int64_t)k * kMxBytes;
        for (int i = 0; i < parts; ++i, src += (int64_t)g.stages * kMxBytes) {
          bulk_g2s(stage + kMxBytes + i * kMxCodes, src + at.sub * 128, min(codes - i * kMxCodes, (uint32_t)kMxCodes), bar, keep);
          bulk_g2s(stage + kMxBytes + C::kXCodes + i * 1024, src + kMxCodes, 1024, bar, keep);
        }
      };
      int k = k0;
      if (!waited) {  // the weights of the first stages do not depend on the preceding kernel
        const int ahead = min(S, k1 - k0);
        if (elect_one())
          for (int i = 0; i < ahead; ++i) {
            const uint32_t bar = smem_addr(&b_full[i]);
            mbar_expect_tx(bar, bytes);
            bulk_g2s(ring + i * C::kStageBytes, w + (int64_t)(k0 + i) * kMxBytes, kMxBytes, bar, w_policy);
          }
        asm volatile("griddepcontrol.wait;" ::: "memory");
        waited = true;
        if (elect_one())
          for (int i = 0; i < ahead; ++i) copy_x(ring + i * C::kStageBytes, smem_addr(&b_full[i]), k0 + i);
        it = ahead, k = k0 + ahead;
      }
      for (; k < k1; ++k, ++it) {
        const uint32_t s = it % S, bar = smem_addr(&b_full[s]), stage = ring + s * C::kStageBytes;
        if (it >= S && !wait_warp(&b_empty[s], it / S - 1)) break;
        if (elect_one()) {
          mbar_expect_tx(bar, bytes);
          bulk_g2s(stage, w + (int64_t)k * kMxBytes, kMxBytes, bar, w_policy);
          copy_x(stage, bar, k);
        }
        __syncwarp();
      }
    } else if (warp == 1) {
      const uint32_t buf = tile_count & 1, acc = tmem + buf * C::kSecond;
      // 256 columns: the previous tile's epilogue has read the columns that both share; else: the last but one is done
      if (TN == 256 ? tile_count >= 1 : tile_count >= 2) {
        const uint32_t before = tile_count - (TN == 256 ? 1 : 2);
        wait_warp(&b_free[before & 1], before >> 1);
      }
      tc::fence_after();
      const int n = (at.n + 15) & ~15;
      const uint32_t desc[2] = {instr_desc_mxf4(n, 0), instr_desc_mxf4(n, 1)};
      const uint32_t column = TN == 64 ? (uint32_t)at.sub >> 5 : 0;  // where the tile's scales begin: 0 or 2
      for (int k = k0; k < k1; ++k, ++it) {
        const uint32_t s = it % S, stage = ring + s * C::kStageBytes;
        if (!wait_warp(&b_full[s], it / S)) break;
        tc::fence_after();
        if (elect_one()) {
          const uint32_t sw = tmem + C::kScaleCol + (it & 1) * C::kScaleSet, sx = sw + 8;
          const uint32_t x_scales = stage + kMxBytes + C::kXCodes;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            copy_scales(sw + 4 * h, stage + kMxCodes + h * 512);
#pragma unroll
            for (int i = 0; i < C::kParts; ++i)
              copy_scales(sx + (h * C::kParts + i) * 4, x_scales + i * 1024 + h * 512);
          }
          const uint64_t da = desc_swizzled(stage), db = desc_swizzled(stage + kMxBytes);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_mxf4(acc, da + j * 2, db + j * 2, desc[j & 1], sw + (j >> 1) * 4, sx + (j >> 1) * 4 * C::kParts + column,
                     k > k0 || j > 0);
          tc::mma_commit(smem_addr(&b_empty[s]));
          if (k == k1 - 1) tc::mma_commit(smem_addr(&b_acc[buf]));
        }
        __syncwarp();
      }
    } else {
      const uint32_t buf = tile_count & 1, lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t acc = tmem + lanes + buf * C::kSecond;
      const int in = (warp & 3) * 32 + lane, n = at.rt * kMxRows + in;
      wait_warp(&b_acc[buf], tile_count >> 1);
      tc::fence_after();
      if (ok) {
        // in the order in which the next tile's products need the columns: the first accumulator's last 64 first
        for (int i = 0; i < TN / 32; ++i) {
          const int c0 = ((TN == 256 && buf == 0) ? (i + 6) % 8 : i) * 32;
          uint32_t v[2][16];
          if (c0 < at.n) {
            load_columns(acc + c0, v[0], v[1]);
          }
          if (!SPLIT && i == (TN == 256 ? 1 : TN / 32 - 1)) {
            tc::fence_before();
            arrive_bar(smem_addr(&b_free[buf]));
          }
          if (c0 < at.n) {
            if constexpr (SPLIT) {  // into the ring: all of its stages have been multiplied
              const uint32_t mine = ring + (c0 * 128 + in) * 4;
#pragma unroll
              for (int c = 0; c < 32; ++c)
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(mine + c * 512), "r"(v[c >> 4][c & 15]) : "memory");
            } else if (n < g.N) {
              with_type(g.y, g.dtype, [&](auto* y) {
                auto* to = y + (int64_t)(at.row0 + c0) * g.ldy + n;
                if (c0 + 32 <= at.n) {
#pragma unroll
                  for (int c = 0; c < 32; ++c, to += g.ldy) store_one(to, __uint_as_float(v[c >> 4][c & 15]));
                } else {
#pragma unroll
                  for (int c = 0; c < 32; ++c, to += g.ldy)
                    if (c0 + c < at.n) store_one(to, __uint_as_float(v[c >> 4][c & 15]));
                }
              });
            }
          }
        }
      }
      if (SPLIT) {
        tc::fence_before();
        arrive_bar(smem_addr(&b_free[buf]));
      }
    }
    ++tile_count;
    if constexpr (SPLIT) {
      cluster_sync();
      if (warp >= 2) {
        const int in = (warp - 2) * 32 + lane, n = at.rt * kMxRows + in;
        const int c1 = (int)(at.n * (rank + 1) / ranks);
        for (int c = (int)(at.n * rank / ranks); c < c1; c += 8) {  // eight columns' loads are under way at a time
          float sum[8] = {};
          for (uint32_t r = 0; r < ranks; ++r) {
            float part[8];
            uint32_t there;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(ring + (c * 128 + in) * 4), "r"(r));
#pragma unroll
            for (int i = 0; i < 8; ++i)  // (past the last column: inside the ring still)
              asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part[i]) : "r"(there + i * 512) : "memory");
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += part[i];
          }
          if (n < g.N && !s_abort)
            with_type(g.y, g.dtype, [&](auto* y) {
              auto* to = y + (int64_t)(at.row0 + c) * g.ldy + n;
#pragma unroll
              for (int i = 0; i < 8; ++i, to += g.ldy)
                if (c + i < c1) store_one(to, sum[i]);
            });
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the ring's next stages come through the other proxy
      cluster_sync();
    }
  }

  // Nothing of this CTA's is under way when it ends: the epilogue has seen the last products, and so the last copies, unless a
  // wait ran out.
  if (warp == 0 && !waited) asm volatile("griddepcontrol.wait;" ::: "memory");
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (s_abort) {
    if (threadIdx.x == 0) {
      atomicCAS(&g_device_error, 0, kErrTimeout);
      for (uint32_t i = it > S ? it - S : 0; i < it; ++i) mbar_wait(smem_addr(&b_full[i % S]), (i / S) & 1, kWaitLimit);
    }
    if (warp == 1) {  // (a commit is for the products of the lane that makes it: the one that is elected for them)
      if (elect_one()) tc::mma_commit(smem_addr(&b_end));
      __syncwarp();
      mbar_wait(smem_addr(&b_end), 0, kWaitLimit);
    }
    __syncthreads();
  }
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

template <int TN, bool SPLIT>
int launch_tile(const MxGemm& g, int ctas, int ranks, cudaStream_t stream) {
  using C = MxTile<TN>;
  const int smem = C::kSmem + (g.offsets ? (g.experts + 1) * 12 : 0);
  static std::atomic<unsigned long long> done{0};  // devices on which the kernel may take that much
  const auto kernel = mx_gemm_kernel<TN, SPLIT>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1))) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem + (kMaxExperts + 1) * 12);
    if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return fail(B2Q_ECUDA, "mx_gemm: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ctas * ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ranks, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = SPLIT ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, g);
  return after_launch("mx_gemm");
}

}  // namespace

// Rows of x a tile, and CTAs that share its K.
struct Shape {
  int tn, ranks;
};

// The shape that takes least time by what rounds of tiles take, us. Measured on layers of 1000 to 14336 rows, K of 1024 to 8192,
// with 16 to 2048 rows of x and all shapes: a stage of a tile with n rows takes 0.28 (n = 64), 0.33 (128), 0.45 (256); its
// epilogue 2, 2.6, 4, beside the next tile's products; joining parts of K 1 + n / 50. Chosen / the next best, us: 8192 x 8192 with 64
// rows 13.3 (K in 2) / 15.1 (whole), with 256 rows 17.2 (128 a tile) / 19.5 (256), with 512 rows 21.2 (256) / 30.7 (128); 4096 x
// 4096 with 256 rows 10.2 (64) / 11.2 (128). Clusters of 8 wait for as many free SMs of a kind: 2048 x 8192 with 16 rows 14.8, K in 4
// parts 8.4.
// Experts: by the average, so that no size has to be known on the host. 4096 tokens, 4 of 32 experts of 4096 x 4096, with at the most
// 578 / 2754 / 4029 rows an expert: 154 / 158 / 150 us; 512 tokens with 84 / 173 / 512: 69 / 73 / 63.
static Shape choose_shape(int64_t used, int64_t each, int64_t row_tiles, int64_t stages, int sms) {
  Shape best = {64, 1};
  double least = 1e30;
  for (int tn : {64, 128, 256})
    for (int ranks : {1, 2, 4}) {
      const int64_t tiles = used * ((each + tn - 1) / tn) * row_tiles;
      if (ranks > 1 && (tn == 256 || tiles * ranks > sms || stages < 2 * ranks)) continue;
      const double n = (double)std::min<int64_t>(each, tn);
      const double stage = n <= 64 ? 0.28 : n <= 128 ? 0.28 + (n - 64) * 0.0008 : 0.33 + (n - 128) * 0.00094;
      const double work = (double)((stages + ranks - 1) / ranks) * stage, after = 1.3 + n / 96;
      const double rounds = (double)((tiles + sms / ranks - 1) / (sms / ranks));
      const double time = (rounds - 1) * std::max(work, after) + work + after + (ranks > 1 ? 1 + n / 50 : 0);
      if (time < least) least = time, best = {tn, ranks};
    }
  return best;
}

int launch_mx_gemm(const MxGemm& g, cudaStream_t stream) {
  if (g.rows == 0 || g.N == 0) return B2Q_OK;
  DeviceInfo dev;
  int rc = device_info(&dev);
  if (rc) return rc;
  // rows an expert has on average, of the experts that can have any
  const int64_t used = g.offsets ? std::min<int64_t>(g.experts, g.rows) : 1;
  const int64_t each = (g.rows + used - 1) / used;
  const Shape shape = choose_shape(used, each, g.row_tiles, g.stages, dev.sms);
  const int tn = shape.tn, ranks = shape.ranks;
  // every tile that there can be: each expert's last one may be all but empty
  const int64_t most = ((g.rows + tn - 1) / tn + (g.offsets ? used : 0)) * g.row_tiles;
  if (most > INT32_MAX / 2) return fail(B2Q_ERANGE, "mx_gemm: too many tiles");
  const int ctas = (int)std::min<int64_t>(most, dev.sms / ranks);
  switch (tn) {
    case 64: return ranks > 1 ? launch_tile<64, true>(g, ctas, ranks, stream) : launch_tile<64, false>(g, ctas, 1, stream);
    case 128: return ranks > 1 ? launch_tile<128, true>(g, ctas, ranks, stream) : launch_tile<128, false>(g, ctas, 1, stream);
    default: return launch_tile<256, false>(g, ctas, 1, stream);
  }
}

int mx_gemm_error(int* code, int clear) { return read_error_word(g_device_error, code, clear); }

static int check_out(const char* who, int dtype, const void* y, int64_t ldy, int64_t rows, int64_t N) {
  if (dtype < B2Q_DTYPE_F32 || dtype > B2Q_DTYPE_BF16) return fail(B2Q_EINVAL, "%s: y: unknown dtype %d", who, dtype);
  if (!y) return fail(B2Q_EINVAL, "%s: y is NULL", who);
  if (rows > 1 && ldy < N) return fail(B2Q_EINVAL, "%s: y: row stride %lld < %lld", who, (long long)ldy, (long long)N);
  if (!aligned(y, mx_dtype_size(dtype))) return fail(B2Q_EALIGN, "%s: y is not aligned to its type", who);
  return B2Q_OK;
}

static int check_weights(const char* who, const uint8_t* w, int64_t N) {
  if (!w) return fail(B2Q_EINVAL, "%s: w is NULL", who);
  if (N > INT32_MAX - 128) return fail(B2Q_ERANGE, "%s: N=%lld", who, (long long)N);
  if (!aligned(w, 128)) return fail(B2Q_EALIGN, "%s: w must be 128-byte aligned", who);
  return B2Q_OK;
}

}  // namespace b2q

using namespace b2q;

extern "C" {

int b2q_mx_matmul(const uint8_t* a, const uint8_t* w, int64_t M, int64_t N, int64_t K, int dtype, void* y, int64_t ldy,
                  b2q_stream_t stream) {
  const char* who = "b2q_mx_matmul";
  int rc = check_mx_shape(who, M, K);
  if (!rc) rc = check_mx_shape(who, N, K);
  if (rc || M == 0 || N == 0) return rc;
  rc = check_weights(who, w, N);
  if (!rc) rc = check_out(who, dtype, y, ldy, M, N);
  if (rc) return rc;
  if (!a) return fail(B2Q_EINVAL, "%s: a is NULL", who);
  if (!aligned(a, 128)) return fail(B2Q_EALIGN, "%s: a must be 128-byte aligned", who);
  const MxGemm g = {w, a, y, nullptr, nullptr, ldy, M, (int)N, (int)mx_tiles(N), (int)mx_stages(K), 1, dtype, 0};
  return launch_mx_gemm(g, stream);
}

size_t b2q_mx_linear_workspace_size(int64_t M, int64_t N, int64_t K) {
  if (check_mx_shape("b2q_mx_linear_workspace_size", M, K) || check_mx_shape("b2q_mx_linear_workspace_size", N, K)) return 0;
  return mx_gemv_takes(M, 1, 1, N, K) ? 0 : b2q_mx_bytes(1, M, K);
}

int b2q_mx_linear(const b2q_mx_linear_args* args, b2q_stream_t stream) {
  const char* who = "b2q_mx_linear";
  if (!args) return fail(B2Q_EINVAL, "%s: null arguments", who);
  const auto [x, w, y, workspace, ldx, M, N, K, ldy, workspace_bytes, x_dtype, dtype] = *args;
  int rc = check_mx_shape(who, M, K);
  if (!rc) rc = check_mx_shape(who, N, K);
  if (!rc) rc = check_mx_rows(who, "x", x_dtype, x, ldx, M, K);
  if (rc || M == 0 || N == 0) return rc;
  rc = check_weights(who, w, N);
  if (!rc) rc = check_out(who, dtype, y, ldy, M, N);
  if (rc) return rc;
  if (!aligned(x, 16) || (M > 1 && ldx * mx_dtype_size(x_dtype) % 16))
    return fail(B2Q_EALIGN, "%s: x and its row stride must be 16-byte aligned", who);
  if (mx_gemv_takes(M, 1, 1, N, K))
    return launch_mx_gemv({w, x, y, nullptr, nullptr, ldx, ldy, M, 1, 1, N, K, x_dtype, dtype, 0}, stream);
  const size_t need = b2q_mx_bytes(1, M, K);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 128))
    return fail(B2Q_EINVAL, "%s: workspace of %zu bytes, 128-byte aligned, needed (%zu given)", who, need, workspace_bytes);
  uint8_t* image = static_cast<uint8_t*>(workspace);
  rc = launch_mx_quantize(x_dtype, x, ldx, M, M, K, image, nullptr, 1, stream);
  if (rc) return rc;
  const MxGemm g = {w, image, y, nullptr, nullptr, ldy, M, (int)N, (int)mx_tiles(N), (int)mx_stages(K), 1, dtype, 1};
  return launch_mx_gemm(g, stream);
}

}  // extern "C"
