// Experts: the router's choice, the tokens' choices sorted by expert, and the experts' rows brought back.
//
// Route: a warp a token, the logits in registers as whole numbers in the logits' order (0: masked or NaN); the largest is one
// warp-wide maximum, the lowest index that has it a minimum (16-bit logits: the same maximum), k times. 16384 tokens of 256
// experts, 8 choices: some 600 instructions a token, whose issue takes 14 of 27 us; placing them 9.
//
// Sort: stable, by counting. The choices (token * top + j) are cut into runs, one a warp; a warp counts its run's experts 32
// choices at a time (lanes with the same expert find each other with one match), the counts before each warp's run give
// every choice its place, and a second walk over the run hands the places out. A short list is one launch: a cluster routes
// it and its first CTA, to which the others send their choices, places it. A long one is two: CTAs all over the GPU route and
// count their tokens, then each adds up what the others before it counted and places its own. The order is always the same.
//
// Combine: a thread adds the same 32 bytes of a token's rows, in order of its choices, in f32: one pass, bound by memory
// (65536 rows of 4096 bf16: 99 us, 6.1 TB/s).
#include <algorithm>
#include <atomic>

#include "mx_device.cuh"

namespace b2q {

namespace {

constexpr int64_t kMostChoices = 1 << 26, kMostPart = 14000;  // in a plan; in a part, whose experts lie in shared memory
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kRun = 64;  // choices a warp counts, and places, at the least
// Lists of up to so many are sorted by one CTA, and routed by its cluster: 1024 choices 5.5 us, 4000 12.7; by two launches 7.
constexpr int kSmallChoices = 1024, kSmallTokens = 128;

struct PlanOut {
  int32_t *offsets, *tiles;            // [experts + 1]
  int32_t *pos, *order;                // [choices]
  int32_t *dest, *dest_row;            // [choices] rows of the operand image: by choice, by sorted row
  int32_t* counts;                     // [parts][experts] of a long list's parts
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// Whole numbers in the order of the logits; 0 for -inf and NaN, which are never chosen. 16-bit logits leave the low 13 bits
// of theirs free (zeros, or ones below 0): there the number of the expert goes, the lowest highest, so that one maximum finds both.
template <typename T>
__device__ __forceinline__ uint32_t order_key(T logit, int e) {
  const float x = to_float(logit) + 0.f;  // -0 as 0
  if (!(x > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(x), k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return sizeof(T) == 4 ? k : (k & 0xffffe000u) | (uint32_t)(0x1fff - e);
}
template <typename T>
__device__ __forceinline__ float key_value(uint32_t k) {
  const bool negative = !(k & 0x80000000u);
  if (sizeof(T) == 2) k = negative ? k | 0x1fffu : k & 0xffffe000u;
  return __uint_as_float(negative ? ~k : k ^ 0x80000000u);
}
// exp(v - top): the largest counts 1, infinities among them
__device__ __forceinline__ float exp_below(float v, float top) { return v == top ? 1.f : expf(v - top); }

// One token by a warp: lane j < top gets the j-th expert (or -1) and its weight.
template <int V, typename T>
__device__ __forceinline__ void route_token(const T* logits, int experts, int top, bool normalize, int lane, int* id, float* weight) {
  uint32_t key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 32 + lane;
    key[v] = e < experts ? order_key(logits[e], e) : 0;
  }
  uint32_t mine = key[0];  // the lane's largest, and (f32) which it is
  int at = 0;
  auto largest_of_lane = [&] {
    mine = key[0], at = 0;
#pragma unroll
    for (int v = 1; v < V; ++v) {
      if constexpr (sizeof(T) == 2) {
        mine = max(mine, key[v]);
      } else {
        if (key[v] > mine) mine = key[v], at = v;
      }
    }
  };
  largest_of_lane();
  uint32_t m = __reduce_max_sync(0xffffffffu, mine);
  const float largest = key_value<T>(m);
  float total = 0.f;
  if (!normalize) {
#pragma unroll
    for (int v = 0; v < V; ++v) total += key[v] ? exp_below(key_value<T>(key[v]), largest) : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  int chosen = -1;
  uint32_t chosen_key = 0;
  for (int j = 0; j < top && m != 0; ++j) {
    int e;
    if (sizeof(T) == 2) {
      e = 0x1fff - (int)(m & 0x1fffu);
    } else {
      e = (int)__reduce_min_sync(0xffffffffu, mine == m ? (uint32_t)(at * 32 + lane) : 0xffffffffu);
    }
    if (lane == j) chosen = e, chosen_key = m;
    if ((e & 31) == lane) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (sizeof(T) == 2 ? key[v] == m : v == at) key[v] = 0;  // (16-bit: no key is there twice)
      largest_of_lane();
    }
    if (j + 1 < top) m = __reduce_max_sync(0xffffffffu, mine);
  }
  const float w = chosen >= 0 ? exp_below(key_value<T>(chosen_key), largest) : 0.f;
  if (normalize) {
    total = w;
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  *id = chosen;
  *weight = chosen >= 0 ? w / total : 0.f;
}

struct RouteArgs {
  const void* logits;
  int64_t ld;
  int top;
  bool normalize;
  int32_t* ids;    // (without routing: given)
  float* weights;
};

// The tokens first, first + step, .. below end by this warp; keep(choice, expert) besides what is stored.
template <int V, typename T, typename Keep>
__device__ __forceinline__ void route_tokens(const RouteArgs& a, int experts, int64_t first, int64_t end, int64_t step, Keep keep) {
  const int lane = threadIdx.x & 31;
  for (int64_t t = first; t < end; t += step) {
    int id;
    float w;
    route_token<V>(static_cast<const T*>(a.logits) + t * a.ld, experts, a.top, a.normalize, lane, &id, &w);
    if (lane < a.top) {
      a.ids[t * a.top + lane] = id, a.weights[t * a.top + lane] = w;
      keep(t * a.top + lane, id);
    }
  }
}

__device__ __forceinline__ uint32_t cluster_address(uint32_t addr, uint32_t rank) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  return there;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_ranks() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// An expert's number, -1 for none.
__device__ __forceinline__ int checked(int id, int experts) {
  if (id >= experts) {
    atomicCAS(&g_device_error, 0, kErrExpert);
    return -1;
  }
  return id < 0 ? -1 : id;
}

// The sums of `rows` and `tiles` over the threads before this one, and over all.
__device__ __forceinline__ void sums_before(int* rows, int* tiles, uint64_t* scratch, int* all_rows, int* all_tiles) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const uint64_t v = (uint64_t)*tiles << 32 | (uint32_t)*rows;
  uint64_t sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += u;
  }
  if (lane == 31) scratch[warp] = sum;
  __syncthreads();
  uint64_t w = lane < warps ? scratch[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += u;
  }
  const uint64_t all = __shfl_sync(0xffffffffu, w, 31), upto = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  sum += (warp ? upto : 0) - v;
  *rows = (int)(uint32_t)sum, *tiles = (int)(sum >> 32), *all_rows = (int)(uint32_t)all, *all_tiles = (int)(all >> 32);
}

// Hands out the places of the CTA's choices first .. end - 1: `before` and `total` are the expert threadIdx.x's choices in
// earlier parts and in all.  ids(i): choice i's expert or -1. s_count: [warps][experts] zeros, s_move [experts].
template <typename Ids, typename Total>
__device__ __forceinline__ void place(Ids ids, Total total_of, int64_t first, int64_t end, int64_t choices, int experts, int* s_count,
                                      int* s_move, uint64_t* scratch, bool writes_totals, int64_t part, int64_t parts,
                                      const PlanOut& p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, all_warps = blockDim.x >> 5;
  const int warps = min(all_warps, (int)((end - first + kRun - 1) / kRun));  // with runs of their own
  const int64_t run = warps ? ((end - first + warps * 32 - 1) / (warps * 32)) * 32 : 0;
  const int64_t begin = min(end, first + warp * run), stop = warp < warps ? min(end, begin + run) : begin;
  int* mine = s_count + warp * experts;
  for (int64_t i = begin; i < stop; i += 32) {
    const int id = i + lane < stop ? ids(i + lane) : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    if (id >= 0 && lane == __ffs(same) - 1) mine[id] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  const int e = threadIdx.x;
  int before = 0, total = 0;  // this expert's choices in earlier parts, and in all
  int here = 0;
  if (e < experts) {
    for (int w = 0; w < warps; ++w) {
      const int c = s_count[w * experts + e];
      s_count[w * experts + e] = here;
      here += c;
    }
  }
  total_of(e, here, &before, &total);
  int offset = total, tile = (total + kMxRows - 1) / kMxRows, placed, tiles;
  sums_before(&offset, &tile, scratch, &placed, &tiles);
  if (e < experts) {
    if (writes_totals) p.offsets[e] = offset, p.tiles[e] = tile;
    for (int w = 0; w < warps; ++w) s_count[w * experts + e] += offset + before;
    s_move[e] = tile * kMxRows - offset;  // from a sorted row to the image's
  }
  if (writes_totals && threadIdx.x == 0) p.offsets[experts] = placed, p.tiles[experts] = tiles;
  __syncthreads();
  for (int64_t i = begin; i < stop; i += 32) {
    const int64_t c = i + lane;
    const int id = c < stop ? ids(c) : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    int row = -1, image = -1;
    if (id >= 0) row = mine[id] + __popc(same & ((1u << lane) - 1)), image = row + s_move[id];
    __syncwarp();
    if (id >= 0 && lane == __ffs(same) - 1) mine[id] += __popc(same);
    __syncwarp();
    if (c < stop) {
      p.pos[c] = row, p.dest[c] = image;
      if (row >= 0) p.order[row] = (int)c, p.dest_row[row] = image;
    }
  }
  for (int64_t r = placed + part * blockDim.x + threadIdx.x; r < choices; r += parts * blockDim.x)
    p.order[r] = -1, p.dest_row[r] = -1;
}

// A short list. V > 0: the CTAs of a cluster route it (logits of type T); the first of them places it.
template <int V, typename T>
__global__ void __launch_bounds__(kSortThreads, 1)
    sort_small_kernel(const RouteArgs a, int choices, int experts, const PlanOut p) {
  extern __shared__ int s_mem[];  // [choices] ids, [experts] moves, [warps][experts] counts
  __shared__ uint64_t s_scratch[32];
  int *s_ids = s_mem, *s_move = s_ids + choices, *s_count = s_move + experts;
  const int warps = min((int)blockDim.x >> 5, (choices + kRun - 1) / kRun);
  const uint32_t rank = cluster_rank(), ranks = cluster_ranks();
  if (V > 0) cluster_arrive();
  if (rank == 0)
    for (int i = threadIdx.x; i < warps * experts; i += blockDim.x) s_count[i] = 0;
  pdl_wait_then_trigger();
  if constexpr (V > 0) {
    const uint32_t first = cluster_address(smem_addr(s_ids), 0);
    cluster_wait();
    route_tokens<V, T>(a, experts, rank * (blockDim.x >> 5) + (threadIdx.x >> 5), choices / a.top, ranks * (blockDim.x >> 5),
                       [&](int64_t c, int id) {
                         asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(first + (uint32_t)c * 4), "r"(id) : "memory");
                       });
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
  } else {
    for (int i = threadIdx.x; i < choices; i += blockDim.x) s_ids[i] = checked(a.ids[i], experts);
    __syncthreads();
  }
  place([&](int64_t i) { return s_ids[i]; }, [](int, int here, int* before, int* total) { *total = here; }, 0, choices, choices,
        experts, s_count, s_move, s_scratch, true, 0, 1, p);
}

// A long list's parts, `per` tokens each: routed and counted, each by the CTAs of a cluster,
template <int V, typename T>
__global__ void __launch_bounds__(512) sort_count_kernel(const RouteArgs a, int64_t tokens, int per, int experts, const PlanOut p) {
  extern __shared__ int s_count[];  // [experts]
  for (int i = threadIdx.x; i < experts; i += blockDim.x) s_count[i] = 0;
  pdl_wait_then_trigger();
  __syncthreads();
  const uint32_t rank = cluster_rank(), ranks = cluster_ranks();
  const int64_t part = blockIdx.x / ranks, first = part * per, end = min(tokens, first + per);
  auto count = [&](int64_t, int id) {
    if (id >= 0) atomicAdd(&s_count[id], 1);  // (whole numbers: in any order)
  };
  if constexpr (V > 0) {
    route_tokens<V, T>(a, experts, first + rank * (blockDim.x >> 5) + (threadIdx.x >> 5), end, ranks * (blockDim.x >> 5), count);
  } else {
    for (int64_t i = first * a.top + rank * blockDim.x + threadIdx.x; i < end * a.top; i += ranks * blockDim.x)
      count(i, checked(a.ids[i], experts));
  }
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  if (rank == 0)
    for (int e = threadIdx.x; e < experts; e += blockDim.x) {
      int sum = s_count[e];
      for (uint32_t r = 1; r < ranks; ++r) {
        int c;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(c) : "r"(cluster_address(smem_addr(s_count + e), r)) : "memory");
        sum += c;
      }
      p.counts[part * experts + e] = sum;
    }
  __syncwarp();
  cluster_arrive();  // the others' counts are read before they end
  cluster_wait();
}

// then placed. As many threads as experts at the least.
__global__ void __launch_bounds__(kSortThreads, 1)
    sort_place_kernel(const int32_t* ids, int top, int64_t tokens, int per, int experts, const PlanOut p) {
  extern __shared__ int s_mem[];  // [per * top] ids, [experts] moves, earlier and all counts, [warps][experts] counts
  __shared__ uint64_t s_scratch[32];
  int *s_ids = s_mem, *s_move = s_ids + per * top, *s_before = s_move + experts, *s_total = s_before + experts;
  int* s_count = s_total + experts;
  const int64_t first = (int64_t)blockIdx.x * per, end = min(tokens, first + per);
  const int n = (int)(end - first) * top, warps = min((int)blockDim.x >> 5, (n + kRun - 1) / kRun);
  for (int i = threadIdx.x; i < warps * experts; i += blockDim.x) s_count[i] = 0;
  for (int e = threadIdx.x; e < experts; e += blockDim.x) s_before[e] = s_total[e] = 0;
  pdl_wait_then_trigger();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int id = ids[first * top + i];
    s_ids[i] = id < experts ? id : -1;
  }
  __syncthreads();
  // the parts' counts of an expert are added up by as many threads as there are for it
  const int parts = gridDim.x, groups = max(1, (int)blockDim.x / experts), group = threadIdx.x / experts;
  if (group < groups) {
    const int e = threadIdx.x - group * experts;
    int before = 0, total = 0;
#pragma unroll 16
    for (int q = group; q < parts; q += groups) {
      const int c = p.counts[(int64_t)q * experts + e];
      total += c;
      before += q < (int)blockIdx.x ? c : 0;
    }
    atomicAdd(&s_before[e], before), atomicAdd(&s_total[e], total);
  }
  __syncthreads();
  place([&](int64_t i) { return s_ids[i - first * top]; },
        [&](int e, int, int* before, int* total) {
          if (e < experts) *before = s_before[e], *total = s_total[e];
        },
        first * top, end * top, tokens * top, experts, s_count, s_move, s_scratch, blockIdx.x == 0, blockIdx.x, parts, p);
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
    if constexpr (B == 32) {
      asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "l"(p));
    } else if constexpr (B == 16) {
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
    if constexpr (B == 32)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                   "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                   : "memory");
    else if constexpr (B == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
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
  // Rows whose loads are under way together: other warps hide the rest. 65536 rows of 4096 bf16 with 1 / 2 / 4 / 8: 100 / 99 / 109 /
  // 174 us; 16384 of 4096 f32 51 / 57 / 63 / 105.
  constexpr int kAtOnce = sizeof(T) == 4 ? 1 : 2;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = item < (1ll << 32) ? (int64_t)((uint32_t)item / (uint32_t)vectors) : item / vectors;
  if (t >= tokens) return;
  const int c = (int)(item - t * vectors) * V::N;
  float sum[V::N] = {};
  for (int j0 = 0; j0 < top; j0 += kAtOnce) {
    V v[kAtOnce];
    float w[kAtOnce];
    int r[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      r[j] = j0 + j < top ? pos[t * top + j0 + j] : -1;
      if (r[j] >= rows) r[j] = -1;
      if (r[j] >= 0) {
        w[j] = weights ? weights[t * top + j0 + j] : 1.f;
        v[j].load(y + r[j] * ldy + c);
      }
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
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
  const int bytes = all % 32 == 0 ? 32 : all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
  const int64_t vectors = N * (int)sizeof(T) / bytes, grid = (tokens * vectors + 255) / 256;
  if (vectors > INT32_MAX || grid > INT32_MAX) return fail(B2Q_ERANGE, "b2q_experts_combine: too many values for one launch");
  auto launch = [&](auto kernel) {
    launch_maybe_pdl(kernel, dim3((unsigned)grid), dim3(256), 0, stream, static_cast<const T*>(y), ldy, rows, pos, weights, tokens,
                     top, (int)vectors, static_cast<T*>(out), ldo);
  };
  if (bytes == 32) launch(combine_kernel<T, 32>);
  else if (bytes == 16) launch(combine_kernel<T, 16>);
  else if (bytes == 8) launch(combine_kernel<T, 8>);
  else if (bytes == 4) launch(combine_kernel<T, 4>);
  else if constexpr (sizeof(T) == 2) launch(combine_kernel<T, 2>);
  return after_launch("experts_combine");
}

// A long list's parts: tokens each, and how many.
struct Parts {
  int per, count;
};
Parts parts_of(int64_t tokens, int64_t top) {
  // some 1000 choices or 32 tokens each (300 tokens of 128 experts, 8 choices: 9.8 us, 16.4 in parts of 128 tokens), but no more
  // than about fill the GPU: the counts are [parts][experts], and every CTA reads them (16384 tokens of 256: 128 parts 27.3, 144 31.9)
  const int64_t choices = tokens * top;
  const int64_t want = std::max({(int64_t)1, std::min<int64_t>(std::max(choices / 1024, tokens / 32), 128), (choices + kMostPart - 1) / kMostPart});
  const int64_t per = (tokens + want - 1) / want;
  return {(int)per, (int)((tokens + per - 1) / per)};
}

bool is_small(int64_t tokens, int64_t top, bool routed) {
  return tokens * top <= kSmallChoices && (!routed || tokens <= kSmallTokens);
}

// Lets a kernel take up to `most` bytes of shared memory, once a device.
template <typename Kernel>
int allow_smem(Kernel kernel, int most, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1))) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  return e == cudaSuccess ? B2Q_OK : fail(B2Q_ECUDA, "experts: %s", cudaGetErrorString(e));
}

template <typename... KArgs, typename... Args>
int launch_cluster(const char* who, void (*kernel)(KArgs...), int grid, int ranks, int threads, size_t smem, cudaStream_t stream,
                   Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ranks, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
  return after_launch(who);
}

constexpr int kSortSmem = 220 * 1024;
static_assert((kMostPart + kMaxTop + kMaxExperts * (3 + kSortWarps)) * 4 <= kSortSmem, "a part's experts and counts");

template <int V, typename T>
int route_and_sort(const RouteArgs& a, int64_t tokens, int experts, const PlanOut& p, cudaStream_t stream) {
  const int64_t choices = tokens * a.top;
  static std::atomic<unsigned long long> done_small{0}, done_place{0};
  if (is_small(tokens, a.top, V > 0)) {
    // A warp a run and a thread an expert in the CTA that places; routing, a cluster of up to 8 with some 8 tokens each (one
    // CTA takes 64 tokens of 128 experts, 8 choices each, in 7 us, 4 of them the issue of its instructions).
    const int ranks = V == 0 ? 1 : tokens > 32 ? 8 : tokens > 8 ? 4 : 1;
    const int runs = (int)(choices + kRun - 1) / kRun, routing = V > 0 ? (int)(tokens + ranks - 1) / ranks : 8;
    const int threads = std::min(kSortThreads, std::max({runs, routing, (experts + 31) / 32, 1}) * 32);
    const size_t smem = (size_t)(choices + experts + std::min(threads / 32, runs) * experts) * 4;
    int rc = allow_smem(sort_small_kernel<V, T>, kSortSmem, done_small);
    if (rc) return rc;
    return launch_cluster("experts_sort", sort_small_kernel<V, T>, ranks, ranks, threads, smem, stream, a, (int)choices, experts, p);
  }
  const Parts q = parts_of(tokens, a.top);
  const size_t smem_place = ((size_t)q.per * a.top + (size_t)experts * (3 + kSortWarps)) * 4;
  int rc = allow_smem(sort_place_kernel, kSortSmem, done_place);
  if (rc) return rc;
  const int ranks = V > 0 ? 4 : 1;
  rc = launch_cluster("experts_count", sort_count_kernel<V, T>, q.count * ranks, ranks, 512, (size_t)experts * 4, stream, a, tokens, q.per,
                      experts, p);
  if (rc) return rc;
  launch_maybe_pdl(sort_place_kernel, dim3(q.count), dim3(kSortThreads), smem_place, stream, a.ids, a.top, tokens, q.per, experts, p);
  return after_launch("experts_sort");
}

template <typename T>
int route_typed(const RouteArgs& a, int64_t tokens, int experts, const PlanOut& p, cudaStream_t stream) {
  if (experts <= 32) return route_and_sort<1, T>(a, tokens, experts, p, stream);
  if (experts <= 64) return route_and_sort<2, T>(a, tokens, experts, p, stream);
  if (experts <= 128) return route_and_sort<4, T>(a, tokens, experts, p, stream);
  if (experts <= 256) return route_and_sort<8, T>(a, tokens, experts, p, stream);
  if (experts <= 512) return route_and_sort<16, T>(a, tokens, experts, p, stream);
  return route_and_sort<32, T>(a, tokens, experts, p, stream);
}

// The plan's parts in its one allocation: offsets, tiles [experts + 1 each]; pos, order, dest, dest_row [choices each]; counts.
PlanOut plan_parts(int32_t* plan, int64_t choices, int64_t experts) {
  int32_t* lists = plan + 2 * (experts + 1);
  return {plan, plan + experts + 1, lists, lists + choices, lists + 2 * choices, lists + 3 * choices, lists + 4 * choices};
}

int check_plan(const char* who, const int32_t* plan, int64_t tokens, int64_t top, int64_t experts) {
  if (tokens < 0 || top < 1 || top > kMaxTop)
    return fail(B2Q_EINVAL, "%s: %lld tokens, %lld choices each (1..%lld)", who, (long long)tokens, (long long)top, (long long)kMaxTop);
  if (experts < 1 || experts > kMaxExperts)
    return fail(B2Q_EINVAL, "%s: %lld experts (1..%lld)", who, (long long)experts, (long long)kMaxExperts);
  if (tokens > kMostChoices / top) return fail(B2Q_ERANGE, "%s: %lld tokens of %lld choices", who, (long long)tokens, (long long)top);
  if (!plan) return fail(B2Q_EINVAL, "%s: plan is NULL", who);
  if (!aligned(plan, 4)) return fail(B2Q_EALIGN, "%s: plan must be 4-byte aligned", who);
  return B2Q_OK;
}

}  // namespace

int experts_error(int* code, int clear) { return read_error_word(g_device_error, code, clear); }

}  // namespace b2q

using namespace b2q;

extern "C" {

size_t b2q_experts_plan_words(int64_t tokens, int64_t top, int64_t experts) {
  int32_t any = 0;
  if (check_plan("b2q_experts_plan_words", &any, tokens, top, experts)) return 0;
  const int64_t choices = tokens * top;
  return (size_t)(2 * (experts + 1) + 4 * choices + (is_small(tokens, top, true) ? 0 : parts_of(tokens, top).count * experts));
}

int b2q_experts_route(const b2q_experts_route_args* args, b2q_stream_t stream) {
  const char* who = "b2q_experts_route";
  if (!args) return fail(B2Q_EINVAL, "%s: null arguments", who);
  const auto [logits, ids, weights, plan, ld, tokens, experts, top, dtype, normalize] = *args;
  int rc = check_plan(who, plan, tokens, top, experts);
  if (rc) return rc;
  if (dtype < B2Q_DTYPE_F32 || dtype > B2Q_DTYPE_BF16) return fail(B2Q_EINVAL, "%s: unknown dtype %d", who, dtype);
  if (top > experts) return fail(B2Q_EINVAL, "%s: %lld choices of %lld experts", who, (long long)top, (long long)experts);
  if (tokens > 0 && (!logits || !ids || !weights)) return fail(B2Q_EINVAL, "%s: null pointer", who);
  if (tokens > 1 && ld < experts) return fail(B2Q_EINVAL, "%s: row stride %lld < %lld", who, (long long)ld, (long long)experts);
  if (!aligned(logits, mx_dtype_size(dtype)) || !aligned(ids, 4) || !aligned(weights, 4))
    return fail(B2Q_EALIGN, "%s: a pointer is not aligned to its type", who);
  const PlanOut p = plan_parts(plan, tokens * top, experts);
  const RouteArgs a = {logits, ld, (int)top, normalize != 0, ids, weights};
  if (dtype == B2Q_DTYPE_F32) return route_typed<float>(a, tokens, (int)experts, p, stream);
  if (dtype == B2Q_DTYPE_F16) return route_typed<__half>(a, tokens, (int)experts, p, stream);
  return route_typed<__nv_bfloat16>(a, tokens, (int)experts, p, stream);
}

int b2q_experts_sort(const int32_t* ids, int64_t tokens, int64_t top, int64_t experts, int32_t* plan, b2q_stream_t stream) {
  const char* who = "b2q_experts_sort";
  int rc = check_plan(who, plan, tokens, top, experts);
  if (rc) return rc;
  if (tokens > 0 && !ids) return fail(B2Q_EINVAL, "%s: ids is NULL", who);
  if (!aligned(ids, 4)) return fail(B2Q_EALIGN, "%s: ids must be 4-byte aligned", who);
  const RouteArgs a = {nullptr, 0, (int)top, false, const_cast<int32_t*>(ids), nullptr};
  return route_and_sort<0, float>(a, tokens, (int)experts, plan_parts(plan, tokens * top, experts), stream);
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

int b2q_experts_linear(const b2q_experts_linear_args* args, b2q_stream_t stream) {
  const char* who = "b2q_experts_linear";
  if (!args) return fail(B2Q_EINVAL, "%s: null arguments", who);
  const auto [x, w, plan, y, workspace, ldx, tokens, top, experts, N, K, ldy, workspace_bytes, x_dtype, dtype, gather] = *args;
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
  rc = launch_mx_quantize(x_dtype, x, ldx, rows, rows, K, image, gather ? p.dest : p.dest_row, gather ? (int)top : 1, stream);
  if (rc) return rc;
  const MxGemm g = {w, image, y, p.offsets, p.tiles, ldy, choices, (int)N, (int)mx_tiles(N), (int)mx_stages(K), (int)experts,
                    dtype, 1};
  return launch_mx_gemm(g, stream);
}

int b2q_experts_combine(const b2q_experts_combine_args* args, b2q_stream_t stream) {
  const char* who = "b2q_experts_combine";
  if (!args) return fail(B2Q_EINVAL, "%s: null arguments", who);
  const auto [y, plan, weights, out, ldy, tokens, top, experts, N, ldo, dtype] = *args;
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
