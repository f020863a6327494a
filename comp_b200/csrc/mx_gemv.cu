// MXFP4 products of up to 4 rows (the next tokens of a few sequences), quantizing the rows on the way: one launch.
//
// What counts here is the stream of weights, 17/32 byte a value, and what a launch costs before and after it. As in mx_gemm.cu
// a CTA's tile is 128 weight rows, whose stages of 256 values of K one thread copies into a ring and another one multiplies;
// but all rows of x stay in shared memory, and their scales in tensor memory, for as long as the CTA lives: eight warps quantize
// them there while the first weights are on their way. (Asking for those to be brought into L2 before waiting for the
// preceding kernel, a hint that could do no harm, was 1.2 us slower at 8192 x 8192.)
//
// Every CTA reads all rows as they are given, four times the bytes of their codes, from the same lines of L2: 0.5 us a row.
// Measured with 1 / 2 / 4 rows against quantizing first and multiplying then (5 rows; 16 take 0.1 more), us, weights from memory:
// 8192 x 8192 9.2 / 10.1 / 11.3 and 11.6; 14336 x 4096 8.4 / 9.2 / 10.1 and 10.2; 4096 x 14336 8.4 / 9.4 / 10.4 and 11.4; 4096 x 4096
// 4.9 / 5.1 / 5.3 and 7.2; 2000 x 1024 3.4 / 3.6 / 3.8 and 4.9. So up to 4: at 0.5 us a row wide layers are worse off with more.
//
// A layer of experts needs no gathering: every expert that has rows is multiplied with all rows of x (the unit's other side
// is 16 rows at the least), and of the results only those that its choices ask for are stored.
//
// Where there are fewer tiles than SMs the CTAs of a cluster split K: each sends the columns of its part to the CTAs that own
// them (distributed shared memory, counted in bytes by the owner's barrier), which add them in order of rank.
//
// Tensor memory is taken when a CTA begins, and a CTA that finds none free waits for others of its SM, whose kernels may be any.
// A cluster starts as a whole, but nothing says that all of its CTAs find tensor memory. So that calls on several streams cannot
// wait for one another in a ring, no CTA waits for another one of its cluster while it holds tensor memory: each tells the
// others that it has begun before it asks for any, and gives it back as soon as its accumulator is in registers.
#include <algorithm>
#include <atomic>

#include "mx_tc.cuh"

namespace b2q {

namespace {

constexpr int kThreads = 320;                   // copying, multiplying, then 8 warps that quantize, 4 of which store
constexpr int kMaxRing = kGemvRing, kMaxRows = kGemvRows, kXStage = kGemvXStage;
constexpr int kMaxChoices = 128;  // rows of y that a layer of experts makes of them
constexpr uint32_t kScaleW = kGemvScaleW, kScaleX = kGemvScaleX;

struct Gemv {
  const uint8_t* w;
  const void* x;
  void* y;
  const int32_t *offsets, *order;  // of a plan; null: one expert, whose row of y is the row of x
  int64_t ldx, ldy;
  int rows, K, N, row_tiles, stages, experts, choices, dtype;
  int top;      // choices a token where x has a row a token, else 0
  int ring;     // stages of weights in shared memory
  int columns;  // of tensor memory
};

// A tile: its weights, its first column of y, and which rows of y it makes.
struct GemvTile {
  int64_t w_tile;
  int n0, row0, count;
};
__device__ __forceinline__ GemvTile gemv_tile(const Gemv& g, const int* used, const int* offsets, int t) {
  if (!g.offsets) return {t, t * kMxRows, 0, g.rows};
  const int nth = t / g.row_tiles, rt = t - nth * g.row_tiles, e = used[nth], r0 = offsets[nth];
  return {(int64_t)e * g.row_tiles + rt, rt * kMxRows, r0, offsets[nth + 1] - r0};
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) mx_gemv_kernel(const Gemv g) {
  extern __shared__ uint8_t smem_raw[];  // ring [ring][kMxBytes], x codes [stages + 1][kXStage], x scales [stages][512]
  __shared__ uint64_t b_full[kMaxRing], b_empty[kMaxRing], b_acc[2], b_free[2], b_x, b_part, b_end;
  __shared__ float s_part[8][kMxRows];  // the parts of the rows of x whose sums this CTA makes: [row / ranks * ranks + rank]
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_count, s_used[kMaxChoices], s_offsets[kMaxChoices + 1];
  __shared__ uint8_t s_token[kMaxChoices];  // the row of x of each row of y
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank, ranks;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int step = gridDim.x / ranks, start = blockIdx.x / ranks;
  const int k0 = (int)((int64_t)g.stages * rank / ranks), k1 = (int)((int64_t)g.stages * (rank + 1) / ranks), nk = k1 - k0;
  const uint32_t ring = (smem_addr(smem_raw) + 1023) & ~1023u;
  uint8_t* x_mem = smem_raw + (ring - smem_addr(smem_raw)) + g.ring * kMxBytes;
  // (the products read 16 rows: the next stage's for the second half, after the last stage a gap)
  const int x_bytes = (nk + 1) * kXStage;
  const uint32_t x_codes = ring + g.ring * kMxBytes, x_scales = x_codes + x_bytes;

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < g.ring; ++i) mbar_init(smem_addr(&b_full[i]), 1), mbar_init(smem_addr(&b_empty[i]), 1);
    for (int i = 0; i < 2; ++i) mbar_init(smem_addr(&b_acc[i]), 1), mbar_init(smem_addr(&b_free[i]), 128);
    mbar_init(smem_addr(&b_x), 256), mbar_init(smem_addr(&b_part), 1), mbar_init(smem_addr(&b_end), 1);
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  // barriers are ready (waited for before the first parts): told before asking for tensor memory
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)),
                 "r"(g.columns));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (g.offsets && warp == 2) {  // the experts that have rows, and where those begin: 128 experts' loads at a time
    int n = 0;
    for (int e0 = 0; e0 < g.experts; e0 += 128) {
      int at[5];
#pragma unroll
      for (int u = 0; u < 5; ++u) at[u] = g.offsets[min(e0 + u * 32 + lane, g.experts)];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int e = e0 + u * 32 + lane, after = __shfl_down_sync(0xffffffffu, at[u], 1),
                  over = __shfl_sync(0xffffffffu, at[u + 1], 0);
        const int begin = at[u], end = lane < 31 ? after : over;
        const uint32_t some = __ballot_sync(0xffffffffu, end > begin);
        const int i = n + __popc(some & ((1u << lane) - 1));
        if (end > begin && i < kMaxChoices) s_used[i] = e, s_offsets[i] = begin, s_offsets[i + 1] = end;
        n += __popc(some);
      }
    }
    if (lane == 0) s_count = min(n, kMaxChoices);
  } else if (g.offsets && warp == 3) {
    for (int r = lane; r < g.choices; r += 32) s_token[r] = g.top ? max(g.order[r], 0) / g.top : r;  // (-1: nobody's row)
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = s_tmem;
  int tiles = g.offsets ? s_count * g.row_tiles : g.row_tiles;
  if (ranks > 1) tiles = min(tiles, step);  // a cluster has one tile at the most (a plan of other sizes might name more)
  bool ok = true;
  auto wait_warp = [&](uint64_t* bar, uint32_t phase) {
    if (ok) {
      ok = __all_sync(0xffffffffu, mbar_wait(smem_addr(bar), phase & 1, kWaitLimit));
      if (!ok) atomicExch(&s_abort, 1);
    }
    return ok;
  };

  uint32_t issued = 0;  // stages asked for (warp 0)
  if (warp == 0) {
    const uint64_t once = evict_first_policy();
    uint32_t s = 0, round = 0;
    for (int t = start; t < tiles && ok; t += step) {
      const GemvTile at = gemv_tile(g, s_used, s_offsets, t);
      const uint8_t* w = g.w + (at.w_tile * g.stages + k0) * kMxBytes;
      for (int k = 0; k < nk; ++k, w += kMxBytes) {
        if (round && !wait_warp(&b_empty[s], round - 1)) break;
        if (elect_one()) {
          const uint32_t bar = smem_addr(&b_full[s]);
          mbar_expect_tx(bar, kMxBytes);
          bulk_g2s(ring + s * kMxBytes, w, kMxBytes, bar, once);
        }
        __syncwarp();
        ++issued;
        if (++s == (uint32_t)g.ring) s = 0, ++round;
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (start < tiles) {
      const uint32_t desc[2] = {instr_desc_mxf4(16, 0), instr_desc_mxf4(16, 1)};
      wait_warp(&b_x, 0);
      tc::fence_after();
      if (ok && elect_one())
        for (int k = 0; k < nk; ++k) copy_scales(tmem + kScaleX + 4 * k, x_scales + k * 512);
      __syncwarp();
      uint32_t s = 0, round = 0, it = 0, count = 0;
      for (int t = start; t < tiles && ok; t += step, ++count) {
        const uint32_t buf = count & 1, acc = tmem + buf * 16;
        if (count >= 2) wait_warp(&b_free[buf], (count >> 1) - 1);
        tc::fence_after();
        for (int k = 0; k < nk; ++k, ++it) {
          if (!wait_warp(&b_full[s], round)) break;
          tc::fence_after();
          if (elect_one()) {
            const uint32_t stage = ring + s * kMxBytes, sw = tmem + kScaleW + (it & 1) * 8, sx = tmem + kScaleX + 4 * k;
            copy_scales(sw, stage + kMxCodes);
            copy_scales(sw + 4, stage + kMxCodes + 512);
            const uint64_t da = desc_swizzled(stage), db = desc_swizzled(x_codes + k * kXStage);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              mma_mxf4(acc, da + j * 2, db + j * 2, desc[j & 1], sw + (j >> 1) * 4, sx + (j >> 1) * 2, k > 0 || j > 0);
            tc::mma_commit(smem_addr(&b_empty[s]));
            if (k == nk - 1) tc::mma_commit(smem_addr(&b_acc[buf]));
          }
          __syncwarp();
          if (++s == (uint32_t)g.ring) s = 0, ++round;
        }
      }
    }
    __syncwarp();
  } else {
    // quantizing: two threads a block; `per` threads a row, or all for each of several rows at a time
    const int t0 = threadIdx.x - 64, per = nk * 16, together = max(1, 256 / per), mine = per < 256 ? t0 / per : 0;
    const int last = mine < together ? per : 0;
    int in = t0 - mine * per;
    for (int trip = 0; trip < (per + 255) / 256; ++trip, in += 256) {
      const int k = in >> 4, b = (in >> 1) & 7, half = in & 1, at = (k0 + k) * kMxStage + b * 32 + 8 * half;
      for (int r0 = 0; r0 < g.rows; r0 += together) {
        const int row = r0 + mine;
        const bool there = row < g.rows && in < last;
        MxHalf q;
        q.load(static_cast<const T*>(g.x) + row * g.ldx + at, there && at < g.K);
        uint32_t scales = q.finish() << (8 * (b & 3));
        scales |= __shfl_xor_sync(0xffffffffu, scales, 2);
        scales |= __shfl_xor_sync(0xffffffffu, scales, 4);
        if (there) {
          *reinterpret_cast<uint2*>(x_mem + k * kXStage + mx_code_at(row, b) + 8 * half) = q.codes;
          // a stage's scales: row r is lane r, blocks 0..3 in column 0, blocks 4..7 in column 2
          if ((in & 7) == 0) *reinterpret_cast<uint32_t*>(x_mem + x_bytes + k * 512 + row * 16 + (b >> 2) * 8) = scales;
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the tensor cores read them
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&b_x)) : "memory");
  }

  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const bool stores = warp >= 2 && warp < 6;
  // The storing warps have read their last accumulator: tensor memory is given back.
  bool held = true;
  auto give_back = [&] {
    held = false;
    if (stores) {
      tc::fence_before();
      asm volatile("bar.arrive 1, 160;" ::: "memory");
    } else if (warp == 1) {
      asm volatile("bar.sync 1, 160;" ::: "memory");
      tc::fence_after();
      if (__shfl_sync(0xffffffffu, *static_cast<volatile int*>(&s_abort), 0)) {  // products may be under way: they end first
        if (elect_one()) tc::mma_commit(smem_addr(&b_end));
        __syncwarp();
        mbar_wait(smem_addr(&b_end), 0, kWaitLimit);
        __syncwarp();
      }
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(g.columns));
    }
  };
  uint32_t count = 0;
  for (int t = start; t < tiles; t += step, ++count) {  // (once where CTAs share a tile)
    const GemvTile at = gemv_tile(g, s_used, s_offsets, t);
    const int in = (warp & 3) * 32 + lane, n = at.n0 + in;
    uint32_t v[16];
    if (stores) {
      const uint32_t buf = count & 1;
      wait_warp(&b_acc[buf], count >> 1);
      tc::fence_after();
      if (ok) {
        tc::tmem_ld16_nowait(tmem + ((uint32_t)((warp & 3) * 32) << 16) + buf * 16, v);
        tc::tmem_wait_ld_regs(v);
      }
      tc::fence_before();
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&b_free[buf])) : "memory");
    }
    if (ranks == 1) {
      if (stores && ok && n < g.N)
        for (int i = 0; i < at.count; ++i) {
          const int row = at.row0 + i, x_row = g.offsets ? s_token[row] : row;
          uint32_t mine = v[0];
#pragma unroll
          for (int c = 1; c < kMaxRows; ++c) mine = c == x_row ? v[c] : mine;
          store_as(g.y, (int64_t)row * g.ldy + n, g.dtype, __uint_as_float(mine));
        }
      continue;
    }
    // row r of x is summed by CTA r % ranks
    const int owned = (g.rows - (int)rank + (int)ranks - 1) / (int)ranks;
    if (threadIdx.x == 64) mbar_expect_tx(smem_addr(&b_part), (uint32_t)owned * ranks * kMxRows * 4);
    if (stores && ok) {
#pragma unroll
      for (int c = 0; c < kMaxRows; ++c)
        if (c < g.rows) {
          const uint32_t owner = (uint32_t)c % ranks, slot = (uint32_t)c / ranks * ranks + rank;
          uint32_t to, bar;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_addr(&s_part[slot][in])), "r"(owner));
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(smem_addr(&b_part)), "r"(owner));
          asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.u32 [%0], %1, [%2];" ::"r"(to), "r"(v[c]), "r"(bar)
                       : "memory");
        }
    }
    __syncwarp();
    give_back();
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // this CTA has sent its parts
    // Another CTA's parts may be late for as long as other kernels hold the tensor memory that it waits for: a wait that runs out
    // is followed by one for the cluster, after which all have sent theirs.
    bool all_sent = false;
    if (stores && owned > 0 && !__all_sync(0xffffffffu, mbar_wait(smem_addr(&b_part), 0, kWaitLimit))) {
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      all_sent = true;
    }
    if (stores && owned > 0 && wait_warp(&b_part, 0) && n < g.N)
      for (int i = 0; i < owned; ++i) {
        const int x_row = (int)rank + i * (int)ranks;
        float sum = 0.f;
        for (uint32_t r = 0; r < ranks; ++r) sum += s_part[i * ranks + r][in];
        for (int row = at.row0; row < at.row0 + at.count; ++row)
          if ((g.offsets ? s_token[row] : row) == x_row) store_as(g.y, (int64_t)row * g.ldy + n, g.dtype, sum);
      }
    __syncwarp();
    // no CTA ends before all have sent theirs (parts for one that gave up waiting find its memory)
    if (!all_sent) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  __syncwarp();
  if (held) give_back();
  __syncthreads();
  if (s_abort && threadIdx.x == 0) {  // whichever wait ran out: copies that are under way land before the CTA ends
    atomicCAS(&g_device_error, 0, kErrTimeout);
    for (uint32_t i = first_under_way(issued, g.ring); i < issued; ++i)
      mbar_wait(smem_addr(&b_full[i % g.ring]), i / g.ring & 1, kWaitLimit);
  }
}

template <typename T>
int launch_gemv(const Gemv& g, const GemvPlan& p, int ctas, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};  // devices on which the kernel may take all of the shared memory
  const auto kernel = mx_gemv_kernel<T>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1))) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kGemvSmem);
    if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return fail(B2Q_ECUDA, "mx_gemv: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ctas * p.ranks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = p.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.ranks, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kernel, g);
  return after_launch("mx_gemv");
}

}  // namespace

bool mx_gemv_takes(int64_t rows, int64_t choices, int64_t experts, int64_t N, int64_t K) {
  DeviceInfo dev;
  GemvPlan p;
  if (choices > kMaxChoices || device_info(&dev)) return false;
  return plan_gemv(rows, std::min(choices, experts), mx_tiles(N), mx_stages(K), dev.sms, &p);
}

int launch_mx_gemv(const MxGemv& a, cudaStream_t stream) {
  DeviceInfo dev;
  int rc = device_info(&dev);
  if (rc) return rc;
  GemvPlan p;
  const int64_t used = std::min<int64_t>(a.offsets ? a.choices : 1, a.experts), row_tiles = mx_tiles(a.N), stages = mx_stages(a.K);
  if (!plan_gemv(a.rows, used, row_tiles, stages, dev.sms, &p)) return fail(B2Q_ERANGE, "mx_gemv: more rows than the kernel takes");
  const Gemv g = {a.w, a.x, a.y, a.offsets, a.order, a.ldx, a.ldy, (int)a.rows, (int)a.K, (int)a.N, (int)row_tiles, (int)stages,
                  (int)a.experts, (int)a.choices, a.dtype, a.top, p.ring, p.columns};
  // with several CTAs a tile every tile has a cluster of its own
  const int64_t ctas = std::min<int64_t>(used * row_tiles, dev.sms / p.ranks);
  if (a.x_dtype == B2Q_DTYPE_F32) return launch_gemv<float>(g, p, (int)ctas, stream);
  if (a.x_dtype == B2Q_DTYPE_F16) return launch_gemv<__half>(g, p, (int)ctas, stream);
  return launch_gemv<__nv_bfloat16>(g, p, (int)ctas, stream);
}

int mx_gemv_error(int* code, int clear) { return read_error_word(g_device_error, code, clear); }

}  // namespace b2q
