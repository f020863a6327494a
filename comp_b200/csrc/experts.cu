// Experts: the router's choice, the tokens' choices sorted by expert, and the experts' rows brought back.
//
// Route: a warp a token, the logits in registers as whole numbers in the logits' order (0: masked or NaN); the largest is one
// warp-wide maximum, the lowest index that has it a minimum, k times.
//
// Sort: stable, by counting. The choices (token * top + j) are cut into runs, one a warp; a warp counts its run's experts 32
// choices at a time (lanes with the same expert find each other with one match), the counts before each warp's run give
// every choice its place, and a second walk over the run hands the places out. Up to 32 warps are one CTA; longer lists take
// a cluster of 8, which add their counts through distributed shared memory: one launch either way, no atomics, so that the
// order is always the same. A small list's router is the same launch.
//
// Combine: a thread adds the same 16 bytes of a token's rows, in order of its choices, in f32: one pass, bound by memory.
#include <algorithm>
#include <atomic>

#include "mx_device.cuh"

namespace b2q {

namespace {

constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortCluster = 8;

struct PlanOut {
  int32_t *offsets, *tiles;            // [experts + 1]
  int32_t *pos, *order;                // [choices]
  int32_t *dest, *dest_row;            // [choices] rows of the operand image: by choice, by sorted row
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// Whole numbers in the order of the logits; 0 for -inf and NaN, which are never chosen.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 as 0
  if (!(x > -INFINITY)) return 0;
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// exp(v - top): the largest counts 1, infinities among them
__device__ __forceinline__ float exp_below(uint32_t key, uint32_t top) {
  return key == top ? 1.f : expf(key_value(key) - key_value(top));
}

// One token by a warp: lane j < top gets the j-th expert (or -1) and its weight.
template <int V, typename T>
__device__ __forceinline__ void route_token(const T* logits, int experts, int top, bool normalize, int lane, int* id, float* weight) {
  uint32_t key[V];
  uint32_t mine = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 32 + lane;
    key[v] = e < experts ? order_key(to_float(logits[e])) : 0;
    mine = max(mine, key[v]);
  }
  const uint32_t largest = __reduce_max_sync(0xffffffffu, mine);
  float total = 0.f;
  if (!normalize) {
#pragma unroll
    for (int v = 0; v < V; ++v) total += key[v] ? exp_below(key[v], largest) : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  int chosen = -1;
  uint32_t chosen_key = 0;
  for (int j = 0; j < top; ++j) {
    const uint32_t m = j == 0 ? largest : __reduce_max_sync(0xffffffffu, mine);
    if (m == 0) break;
    uint32_t at = 0xffffffffu;
    if (mine == m) {
#pragma unroll
      for (int v = V - 1; v >= 0; --v)
        if (key[v] == m) at = v * 32 + lane;
    }
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == j) chosen = (int)at, chosen_key = m;
    if ((at & 31) == lane) {
      mine = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (v == (int)(at >> 5)) key[v] = 0;
        mine = max(mine, key[v]);
      }
    }
  }
  float w = chosen >= 0 ? exp_below(chosen_key, largest) : 0.f;
  if (normalize) {
    total = w;
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  *id = chosen;
  *weight = chosen >= 0 ? w / total : 0.f;
}

template <int V, typename T>
__device__ __forceinline__ void route_rows(const T* logits, int64_t ld, int64_t tokens, int experts, int top, bool normalize,
                                           int32_t* ids, float* weights, int64_t first, int64_t step) {
  const int lane = threadIdx.x & 31;
  for (int64_t t = first; t < tokens; t += step) {
    int id;
    float w;
    route_token<V>(logits + t * ld, experts, top, normalize, lane, &id, &w);
    if (lane < top) ids[t * top + lane] = id, weights[t * top + lane] = w;
  }
}

template <int V, typename T>
__global__ void __launch_bounds__(256)
    route_kernel(const T* __restrict__ logits, int64_t ld, int64_t tokens, int experts, int top, bool normalize,
                 int32_t* __restrict__ ids, float* __restrict__ weights) {
  pdl_wait_then_trigger();
  route_rows<V>(logits, ld, tokens, experts, top, normalize, ids, weights, (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5),
                (int64_t)gridDim.x * 8);
}

__device__ __forceinline__ int ld_cluster_int(uint32_t addr, uint32_t rank) {
  uint32_t there;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(there) : "memory");
  return v;
}
__device__ __forceinline__ void sync_cluster(uint32_t ranks) {
  if (ranks > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else
    __syncthreads();
}

// The sum of `v` over the threads before this one, and over all (kSortThreads threads).
__device__ __forceinline__ int sum_before(int v, int* scratch, int* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += u;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = sum;
  __syncthreads();
  int w = scratch[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += u;
  }
  *all = __shfl_sync(0xffffffffu, w, 31);
  const int upto = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  return sum - v + (warp ? upto : 0);
}

// V > 0: a single CTA routes first (logits of type T).
template <int V, typename T>
__global__ void __launch_bounds__(kSortThreads, 1)
    sort_kernel(const T* __restrict__ logits, int64_t ld, int top, bool normalize, int32_t* ids, float* weights, int choices,
                int experts, const PlanOut p) {
  extern __shared__ int s_count[];  // [warps][experts], then the CTA's totals [experts]
  __shared__ int s_scratch[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* totals = s_count + kSortWarps * experts;
  uint32_t rank, ranks;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  for (int i = threadIdx.x; i < kSortWarps * experts; i += kSortThreads) s_count[i] = 0;
  pdl_wait_then_trigger();
  if constexpr (V > 0) {
    route_rows<V>(logits, ld, choices / top, experts, top, normalize, ids, weights, warp, kSortWarps);
    __threadfence_block();
  }
  __syncthreads();

  // this warp's run of choices, and what it counts of each expert
  const int run = ((choices + (int)ranks * kSortWarps * 32 - 1) / ((int)ranks * kSortWarps * 32)) * 32;
  const int64_t begin = (int64_t)((int)rank * kSortWarps + warp) * run;
  const int64_t end = min((int64_t)choices, begin + run);
  int* mine = s_count + warp * experts;
  auto expert_of = [&](int64_t i) {
    const int id = i < end ? (V > 0 ? *(volatile const int32_t*)(ids + i) : ids[i]) : -1;
    if (id >= experts) {
      atomicCAS(&g_device_error, 0, kErrExpert);
      return -1;
    }
    return id < 0 ? -1 : id;
  };
  for (int64_t i = begin; i < end; i += 32) {
    const int id = expert_of(i + lane);
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    if (id >= 0 && lane == __ffs(same) - 1) mine[id] += __popc(same);
    __syncwarp();
  }
  __syncthreads();

  // counts before each warp's run; all counts of the CTA
  const int e = threadIdx.x;
  int total = 0;
  if (e < experts) {
    for (int w = 0; w < kSortWarps; ++w) {
      const int c = s_count[w * experts + e];
      s_count[w * experts + e] = total;
      total += c;
    }
    totals[e] = total;
  }
  sync_cluster(ranks);
  int before = 0, all = 0;  // counts of this expert in the CTAs before this one, and in all
  if (e < experts) {
    for (uint32_t r = 0; r < ranks; ++r) {
      const int c = ranks > 1 ? ld_cluster_int(smem_addr(totals + e), r) : total;
      if (r < rank) before += c;
      all += c;
    }
  }
  sync_cluster(ranks);  // the others' totals are read before they change, and before a CTA ends
  int placed, tiles;
  const int offset = sum_before(all, s_scratch, &placed);
  const int tile = sum_before((all + kMxRows - 1) / kMxRows, s_scratch, &tiles);
  if (e < experts) {
    if (rank == 0) p.offsets[e] = offset, p.tiles[e] = tile;
    for (int w = 0; w < kSortWarps; ++w) s_count[w * experts + e] += offset + before;
    totals[e] = tile * kMxRows - offset;  // from a sorted row to the image's
  }
  if (rank == 0 && threadIdx.x == 0) p.offsets[experts] = placed, p.tiles[experts] = tiles;
  __syncthreads();

  for (int64_t i = begin; i < end; i += 32) {
    const int64_t c = i + lane;
    const int id = expert_of(c);
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    int row = -1, image = -1;
    if (id >= 0) row = mine[id] + __popc(same & ((1u << lane) - 1)), image = row + totals[id];
    __syncwarp();
    if (id >= 0 && lane == __ffs(same) - 1) mine[id] += __popc(same);
    __syncwarp();
    if (c < end) {
      p.pos[c] = row, p.dest[c] = image;
      if (row >= 0) p.order[row] = (int)c, p.dest_row[row] = image;
    }
  }
  for (int64_t r = (int64_t)placed + (int)rank * kSortThreads + threadIdx.x; r < choices; r += (int64_t)ranks * kSortThreads)
    p.order[r] = -1, p.dest_row[r] = -1;
}

// Vectors of B bytes of T.
template <typename T, int B>
struct Vec {
  static constexpr int N = B / (int)sizeof(T);
  union {
    T v[N];
    uint32_t w[B >= 4 ? B / 4 : 1];
  };
  __device__ Vec() {}
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (B == 16) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else if constexpr (B == 8) {
      const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = x.x, w[1] = x.y;
    } else if constexpr (B == 4) {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    } else {
      v[0] = *p;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (B == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (B == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else if constexpr (B == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
    else *p = v[0];
  }
};

__device__ __forceinline__ void from_float(float x, float* y) { *y = x; }
__device__ __forceinline__ void from_float(float x, __half* y) { *y = __float2half_rn(x); }
__device__ __forceinline__ void from_float(float x, __nv_bfloat16* y) { *y = __float2bfloat16_rn(x); }

template <typename T, int B>
__global__ void __launch_bounds__(256)
    combine_kernel(const T* __restrict__ y, int64_t ldy, int64_t rows, const int32_t* __restrict__ pos,
                   const float* __restrict__ weights, int64_t tokens, int top, int vectors, T* __restrict__ out, int64_t ldo) {
  pdl_wait_then_trigger();
  using V = Vec<T, B>;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = item < (1ll << 32) ? (int64_t)((uint32_t)item / (uint32_t)vectors) : item / vectors;
  if (t >= tokens) return;
  const int c = (int)(item - t * vectors) * V::N;
  float sum[V::N] = {};
  for (int j0 = 0; j0 < top; j0 += 4) {  // four rows' loads at once
    V v[4];
    float w[4];
    int r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r[j] = j0 + j < top ? pos[t * top + j0 + j] : -1;
      if (r[j] >= rows) r[j] = -1;
      if (r[j] >= 0) {
        w[j] = weights ? weights[t * top + j0 + j] : 1.f;
        v[j].load(y + r[j] * ldy + c);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (r[j] >= 0) {
#pragma unroll
        for (int i = 0; i < V::N; ++i) sum[i] = fmaf(w[j], to_float(v[j].v[i]), sum[i]);
      }
  }
  V o;
#pragma unroll
  for (int i = 0; i < V::N; ++i) from_float(sum[i], &o.v[i]);
  o.store(out + t * ldo + c);
}

template <typename T>
int launch_combine(const void* y, int64_t ldy, int64_t rows, const int32_t* pos, const float* weights, int64_t tokens, int top,
                   int64_t N, void* out, int64_t ldo, cudaStream_t stream) {
  // the widest vectors that both row strides and bases are whole multiples of
  const uint64_t all = (reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(out)) | (uint64_t)(ldy * sizeof(T)) |
                       (uint64_t)(ldo * sizeof(T)) | (uint64_t)(N * sizeof(T));
  const int bytes = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
  const int64_t vectors = N * (int)sizeof(T) / bytes, grid = (tokens * vectors + 255) / 256;
  if (vectors > INT32_MAX || grid > INT32_MAX) return fail(B2Q_ERANGE, "b2q_experts_combine: too many values for one launch");
  auto launch = [&](auto kernel) {
    launch_maybe_pdl(kernel, dim3((unsigned)grid), dim3(256), 0, stream, static_cast<const T*>(y), ldy, rows, pos, weights, tokens,
                     top, (int)vectors, static_cast<T*>(out), ldo);
  };
  if (bytes == 16) launch(combine_kernel<T, 16>);
  else if (bytes == 8) launch(combine_kernel<T, 8>);
  else if (bytes == 4) launch(combine_kernel<T, 4>);
  else if constexpr (sizeof(T) == 2) launch(combine_kernel<T, 2>);
  return after_launch("experts_combine");
}

// Lists of up to so many choices are sorted by one CTA, and routed by it.
constexpr int64_t kSmallChoices = 4096, kSmallTokens = 128;

template <int V, typename T>
int launch_sort(const T* logits, int64_t ld, int top, bool normalize, int32_t* ids, float* weights, int64_t choices, int experts,
                const PlanOut& p, cudaStream_t stream) {
  const auto kernel = sort_kernel<V, T>;
  static std::atomic<unsigned long long> done{0};  // devices on which the kernel may take the memory of the most experts
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1))) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kSortWarps + 1) * (int)kMaxExperts * 4);
    if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return fail(B2Q_ECUDA, "experts_sort: %s", cudaGetErrorString(e));
  const int ranks = choices > kSmallChoices ? kSortCluster : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ranks);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = (size_t)(kSortWarps + 1) * experts * 4;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ranks, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kernel, logits, ld, top, normalize, ids, weights, (int)choices, experts, p);
  return after_launch("experts_sort");
}

template <int V, typename T>
int route_and_sort(const T* logits, int64_t ld, int64_t tokens, int experts, int top, bool normalize, int32_t* ids, float* weights,
                   const PlanOut& p, cudaStream_t stream) {
  const int64_t choices = tokens * top;
  if (tokens <= kSmallTokens) return launch_sort<V>(logits, ld, top, normalize, ids, weights, choices, experts, p, stream);
  DeviceInfo dev;
  int rc = device_info(&dev);
  if (rc) return rc;
  const unsigned grid = (unsigned)std::min<int64_t>((tokens + 7) / 8, (int64_t)dev.sms * 8);
  launch_maybe_pdl(route_kernel<V, T>, dim3(grid), dim3(256), 0, stream, logits, ld, tokens, experts, top, normalize, ids, weights);
  rc = after_launch("experts_route");
  return rc ? rc : launch_sort<0>(static_cast<const float*>(nullptr), 0, top, false, ids, weights, choices, experts, p, stream);
}

template <typename T>
int route_typed(const void* logits, int64_t ld, int64_t tokens, int experts, int top, bool normalize, int32_t* ids, float* weights,
                const PlanOut& p, cudaStream_t stream) {
  const T* x = static_cast<const T*>(logits);
  if (experts <= 32) return route_and_sort<1>(x, ld, tokens, experts, top, normalize, ids, weights, p, stream);
  if (experts <= 64) return route_and_sort<2>(x, ld, tokens, experts, top, normalize, ids, weights, p, stream);
  if (experts <= 128) return route_and_sort<4>(x, ld, tokens, experts, top, normalize, ids, weights, p, stream);
  if (experts <= 256) return route_and_sort<8>(x, ld, tokens, experts, top, normalize, ids, weights, p, stream);
  if (experts <= 512) return route_and_sort<16>(x, ld, tokens, experts, top, normalize, ids, weights, p, stream);
  return route_and_sort<32>(x, ld, tokens, experts, top, normalize, ids, weights, p, stream);
}

// The plan's parts in its one allocation: offsets, tiles [experts + 1 each]; pos, order, dest, dest_row [choices each].
PlanOut plan_parts(int32_t* plan, int64_t choices, int64_t experts) {
  int32_t* lists = plan + 2 * (experts + 1);
  return {plan, plan + experts + 1, lists, lists + choices, lists + 2 * choices, lists + 3 * choices};
}

int check_plan(const char* who, const int32_t* plan, int64_t tokens, int64_t top, int64_t experts) {
  if (tokens < 0 || top < 1 || top > kMaxTop)
    return fail(B2Q_EINVAL, "%s: %lld tokens, %lld choices each (1..%lld)", who, (long long)tokens, (long long)top, (long long)kMaxTop);
  if (experts < 1 || experts > kMaxExperts)
    return fail(B2Q_EINVAL, "%s: %lld experts (1..%lld)", who, (long long)experts, (long long)kMaxExperts);
  if (tokens > (1ll << 30) / top) return fail(B2Q_ERANGE, "%s: %lld tokens of %lld choices", who, (long long)tokens, (long long)top);
  if (!plan) return fail(B2Q_EINVAL, "%s: plan is NULL", who);
  if (!aligned(plan, 4)) return fail(B2Q_EALIGN, "%s: plan must be 4-byte aligned", who);
  return B2Q_OK;
}

}  // namespace

int experts_error(int* code, int clear) { return read_error_word(g_device_error, code, clear); }

}  // namespace b2q

using namespace b2q;

extern "C" {

int b2q_experts_route(int dtype, const void* logits, int64_t ld, int64_t tokens, int64_t experts, int64_t top, int normalize,
                      int32_t* ids, float* weights, int32_t* plan, b2q_stream_t stream) {
  const char* who = "b2q_experts_route";
  int rc = check_plan(who, plan, tokens, top, experts);
  if (rc) return rc;
  if (dtype < B2Q_DTYPE_F32 || dtype > B2Q_DTYPE_BF16) return fail(B2Q_EINVAL, "%s: unknown dtype %d", who, dtype);
  if (top > experts) return fail(B2Q_EINVAL, "%s: %lld choices of %lld experts", who, (long long)top, (long long)experts);
  if (tokens > 0 && (!logits || !ids || !weights)) return fail(B2Q_EINVAL, "%s: null pointer", who);
  if (tokens > 1 && ld < experts) return fail(B2Q_EINVAL, "%s: row stride %lld < %lld", who, (long long)ld, (long long)experts);
  if (!aligned(logits, mx_dtype_size(dtype)) || !aligned(ids, 4) || !aligned(weights, 4))
    return fail(B2Q_EALIGN, "%s: a pointer is not aligned to its type", who);
  const PlanOut p = plan_parts(plan, tokens * top, experts);
  if (dtype == B2Q_DTYPE_F32)
    return route_typed<float>(logits, ld, tokens, (int)experts, (int)top, normalize != 0, ids, weights, p, stream);
  if (dtype == B2Q_DTYPE_F16)
    return route_typed<__half>(logits, ld, tokens, (int)experts, (int)top, normalize != 0, ids, weights, p, stream);
  return route_typed<__nv_bfloat16>(logits, ld, tokens, (int)experts, (int)top, normalize != 0, ids, weights, p, stream);
}

int b2q_experts_sort(const int32_t* ids, int64_t tokens, int64_t top, int64_t experts, int32_t* plan, b2q_stream_t stream) {
  const char* who = "b2q_experts_sort";
  int rc = check_plan(who, plan, tokens, top, experts);
  if (rc) return rc;
  if (tokens > 0 && !ids) return fail(B2Q_EINVAL, "%s: ids is NULL", who);
  if (!aligned(ids, 4)) return fail(B2Q_EALIGN, "%s: ids must be 4-byte aligned", who);
  return launch_sort<0>(static_cast<const float*>(nullptr), 0, (int)top, false, const_cast<int32_t*>(ids), nullptr, tokens * top,
                        (int)experts, plan_parts(plan, tokens * top, experts), stream);
}

size_t b2q_experts_linear_workspace_size(int64_t tokens, int64_t top, int64_t experts, int gather, int64_t N, int64_t K) {
  const char* who = "b2q_experts_linear_workspace_size";
  int32_t any = 0;
  if (check_plan(who, &any, tokens, top, experts) || check_mx_shape(who, N, K)) return 0;
  if (mx_gemv_takes(gather ? tokens : tokens * top, tokens * top, experts, N, K)) return 0;
  // each expert that has rows may leave all but one of its last tile's unused
  const int64_t choices = tokens * top, tiles = choices / kMxRows + std::min(experts, choices);
  return (size_t)tiles * mx_stages(K) * kMxBytes;
}

int b2q_experts_linear(int x_dtype, const void* x, int64_t ldx, int gather, const uint8_t* w, const int32_t* plan, int64_t tokens,
                       int64_t top, int64_t experts, int64_t N, int64_t K, int dtype, void* y, int64_t ldy, void* workspace,
                       size_t workspace_bytes, b2q_stream_t stream) {
  const char* who = "b2q_experts_linear";
  int rc = check_plan(who, plan, tokens, top, experts);
  const int64_t choices = rc ? 0 : tokens * top;
  if (!rc) rc = check_mx_shape(who, N, K);
  const int64_t rows = gather ? tokens : choices;
  if (!rc) rc = check_mx_rows(who, "x", x_dtype, x, ldx, rows, K);
  if (rc || tokens == 0 || N == 0) return rc;
  if (dtype < B2Q_DTYPE_F32 || dtype > B2Q_DTYPE_BF16) return fail(B2Q_EINVAL, "%s: y: unknown dtype %d", who, dtype);
  if (!w || !y) return fail(B2Q_EINVAL, "%s: null pointer", who);
  if (choices > 1 && ldy < N) return fail(B2Q_EINVAL, "%s: y: row stride %lld < %lld", who, (long long)ldy, (long long)N);
  if (N > INT32_MAX - 128) return fail(B2Q_ERANGE, "%s: N=%lld", who, (long long)N);
  if (!aligned(w, 128) || !aligned(y, mx_dtype_size(dtype)) || !aligned(x, 16) ||
      (rows > 1 && ldx * mx_dtype_size(x_dtype) % 16))
    return fail(B2Q_EALIGN, "%s: x and its row stride must be 16-byte aligned, w 128-byte, y to its type", who);
  const PlanOut p = plan_parts(const_cast<int32_t*>(plan), choices, experts);
  if (mx_gemv_takes(rows, choices, experts, N, K))
    return launch_mx_gemv({w, x, y, p.offsets, p.order, ldx, ldy, rows, choices, experts, N, K, x_dtype, dtype,
                           gather ? (int)top : 0}, stream);
  const size_t need = b2q_experts_linear_workspace_size(tokens, top, experts, gather, N, K);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 128))
    return fail(B2Q_EINVAL, "%s: workspace of %zu bytes, 128-byte aligned, needed (%zu given)", who, need, workspace_bytes);
  uint8_t* image = static_cast<uint8_t*>(workspace);
  rc = launch_mx_quantize(x_dtype, x, ldx, rows, K, image, gather ? p.dest : p.dest_row, gather ? (int)top : 1, stream);
  if (rc) return rc;
  const MxGemm g = {w, image, y, p.offsets, p.tiles, ldy, choices, (int)N, (int)mx_tiles(N), (int)mx_stages(K), (int)experts,
                    dtype, 1};
  return launch_mx_gemm(g, stream);
}

int b2q_experts_combine(int dtype, const void* y, int64_t ldy, const int32_t* plan, const float* weights, int64_t tokens,
                        int64_t top, int64_t experts, int64_t N, void* out, int64_t ldo, b2q_stream_t stream) {
  const char* who = "b2q_experts_combine";
  int rc = check_plan(who, plan, tokens, top, experts);
  if (rc) return rc;
  if (dtype < B2Q_DTYPE_F32 || dtype > B2Q_DTYPE_BF16) return fail(B2Q_EINVAL, "%s: unknown dtype %d", who, dtype);
  if (N < 0 || N > INT32_MAX) return fail(B2Q_EINVAL, "%s: N=%lld", who, (long long)N);
  if (tokens == 0 || N == 0) return B2Q_OK;
  if (!y || !out) return fail(B2Q_EINVAL, "%s: null pointer", who);
  if ((tokens * top > 1 && ldy < N) || (tokens > 1 && ldo < N)) return fail(B2Q_EINVAL, "%s: row stride < %lld", who, (long long)N);
  if (!aligned(y, mx_dtype_size(dtype)) || !aligned(out, mx_dtype_size(dtype)) || !aligned(weights, 4))
    return fail(B2Q_EALIGN, "%s: a pointer is not aligned to its type", who);
  const int32_t* pos = plan_parts(const_cast<int32_t*>(plan), tokens * top, experts).pos;
  if (dtype == B2Q_DTYPE_F32)
    return launch_combine<float>(y, ldy, tokens * top, pos, weights, tokens, (int)top, N, out, ldo, stream);
  if (dtype == B2Q_DTYPE_F16)
    return launch_combine<__half>(y, ldy, tokens * top, pos, weights, tokens, (int)top, N, out, ldo, stream);
  return launch_combine<__nv_bfloat16>(y, ldy, tokens * top, pos, weights, tokens, (int)top, N, out, ldo, stream);
}

}  // extern "C"
