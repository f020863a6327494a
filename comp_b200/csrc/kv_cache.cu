// Quantized KV cache: quantizing keys and values into their slots, and reading slots back.
//
// Both are one pass, bound by memory: a write reads the values once and stores 4.5 (q4_0) or 8.5 (q8_0) bits for each, a
// read the reverse. A thread takes quarter l of every 32-value block of a head's row: for q4_0 the values 4l..4l+3 and
// 16+4l..16+4l+3 of a block (the two nibbles of the block's bytes 4l..4l+3), for q8_0 the values 8l..8l+7. In the cache's
// order those are one run of the row, so that a thread's quants are one wide load or store, and four threads' values whole
// 32-byte sectors. (A thread a block's quarter took 195 us for reading 131072 tokens of 8 heads of 128 as bf16: its index
// arithmetic. So 117 us, 5.9 TB/s.) A write of 16384 tokens takes 24 us (3.6 TB/s): its bytes
// are 13 us, and 16 instructions a value (the rounding takes three of them) 15 us of issue, which overlaps with them in part;
// written and read back 65 us at first, 39 us now.
#include <type_traits>

#include "kv_device.cuh"
#include "kv_internal.h"

namespace b2q {

static __device__ int g_kv_error = 0;

// 8 values of a block's quarter l as f32: q4_0 takes two runs of 4, q8_0 one run of 8.
template <int FMT, typename T>
__device__ __forceinline__ void load_quarter(const T* block, int l, float (&v)[8]) {
  if constexpr (FMT == 0) {
    load4(block + 4 * l, *reinterpret_cast<float(*)[4]>(&v[0]));
    load4(block + 16 + 4 * l, *reinterpret_cast<float(*)[4]>(&v[4]));
  } else {
    load4(block + 8 * l, *reinterpret_cast<float(*)[4]>(&v[0]));
    load4(block + 8 * l + 4, *reinterpret_cast<float(*)[4]>(&v[4]));
  }
}

// floor of 0 <= x < 2^23 in the low bits of the result: one addition rounded down, where a conversion would take the unit
// of the special functions.
__device__ __forceinline__ uint32_t floor_bits(float x) { return __float_as_uint(__fadd_rd(x, 8388608.f)); }

// ggml's q4_0 block of 32 values held by 4 consecutive lanes (values 4l.. and 16+4l..): the lane's 4 bytes, f16 d bits.
__device__ __forceinline__ uint32_t quant_q4_0_quarter(const float (&v)[8], int l, uint16_t* d_bits) {
  float hi = v[0], lo = v[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) hi = fmaxf(hi, v[i]), lo = fminf(lo, v[i]);
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
  }
  float m = hi >= -lo ? hi : lo;  // the value of largest magnitude
  if (__any_sync(0xffffffffu, hi == -lo)) {  // both signs have it somewhere in the warp: there the first one counts
    int first = 64;
#pragma unroll
    for (int i = 7; i >= 0; --i)
      if (fabsf(v[i]) == hi) first = 2 * ((i < 4 ? 0 : 12) + 4 * l + i) + (signbit(v[i]) ? 1 : 0);
    first = min(first, __shfl_xor_sync(0xffffffffu, first, 1));
    first = min(first, __shfl_xor_sync(0xffffffffu, first, 2));
    if (hi == -lo) m = (first & 1) ? lo : hi;
  }
  m = __fadd_rn(m, 0.f);  // ggml's maximum begins at +0: a block of zeros, of either sign, has the scale -0
  const float d = __fmul_rn(m, -0.125f);  // m / -8, exact but for underflow
  const float id = d != 0.f ? __fdiv_rn(1.0f, d) : 0.f;
  uint32_t q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = floor_bits(fminf(__fadd_rn(__fmul_rn(v[i], id), 8.5f), 15.5f));  // 0.5 .. 15.5
  *d_bits = __half_as_ushort(__float2half_rn(d));
  return pack_low_bytes(q[0], q[1], q[2], q[3]) | pack_low_bytes(q[4], q[5], q[6], q[7]) << 4;
}

// ggml's q8_0 block, the quants plus 128: the lane's 8 bytes (values 8l..8l+7). roundf(y) is the floor of |y| + 1/2 cut off
// (no sum that is cut off reaches a whole number that it does not hold), with y's sign.
__device__ __forceinline__ uint2 quant_q8_0_quarter(const float (&v)[8], uint16_t* d_bits) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  const float d = __fdiv_rn(amax, 127.0f);
  const float id = d != 0.f ? __fdiv_rn(1.0f, d) : 0.f;
  uint32_t q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = __fmul_rn(v[i], id);
    const uint32_t r = floor_bits(__fadd_rz(fabsf(y), 0.5f));
    q[i] = signbit(y) ? 128u - r : 128u + r;  // the low byte
  }
  *d_bits = __half_as_ushort(__float2half_rn(d));
  return make_uint2(pack_low_bytes(q[0], q[1], q[2], q[3]), pack_low_bytes(q[4], q[5], q[6], q[7]));
}

// N 16-bit words (two to a register) to `dst`, and back, in the widest pieces that N's alignment allows.
template <int N>
__device__ __forceinline__ void store_halves(uint8_t* dst, const uint32_t (&w)[(N + 1) / 2]) {
  if constexpr (N % 8 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; i += 4) *reinterpret_cast<uint4*>(dst + 4 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  } else if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; i += 2) *reinterpret_cast<uint2*>(dst + 4 * i) = make_uint2(w[i], w[i + 1]);
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) *reinterpret_cast<uint32_t*>(dst + 4 * i) = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<uint16_t*>(dst + 2 * i) = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
  }
}
template <int N>
__device__ __forceinline__ void load_halves(const uint8_t* src, uint32_t (&w)[(N + 1) / 2]) {
  if constexpr (N % 8 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(src + 4 * i);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  } else if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; i += 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(src + 4 * i);
      w[i] = v.x, w[i + 1] = v.y;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = *reinterpret_cast<const uint32_t*>(src + 4 * i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t v = *reinterpret_cast<const uint16_t*>(src + 2 * i);
      w[i / 2] = (i & 1) ? (w[i / 2] | v << 16) : v;
    }
  }
}

// A quarter's share of a row, KW 32-bit words: keys as [block][word], values as [unit 2l, 2l + 1][block] of half of that.
// One thread per (token, head, quarter); blockIdx.y 0 = keys, 1 = values.
template <int FMT, int NB, typename T>
__global__ void __launch_bounds__(256)
    kv_write_kernel(const T* __restrict__ k, int64_t k_st, int64_t k_sh, const T* __restrict__ v, int64_t v_st,
                    int64_t v_sh, const int64_t* __restrict__ slots, b2q_kv_cache c, int page_shift, int64_t ntok) {
  pdl_wait_then_trigger();
  constexpr int kRow = NB * (FMT == 0 ? 16 : 32), KW = kRow / 16;
  const bool val = blockIdx.y != 0;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x, r = item >> 2;
  const int l = (int)item & 3;
  const int64_t tok = r < (1u << 31) ? (int64_t)((uint32_t)r / (uint32_t)c.heads) : r / c.heads;
  const int h = (int)(r - tok * c.heads);
  int64_t slot = tok < ntok ? slots[tok] : -1;
  if (slot >= (c.pages << page_shift)) {
    atomicCAS(&g_kv_error, 0, kErrSlot);
    slot = -1;
  }
  // no early return: the four lanes of a row stay together for the shuffles
  float f[NB][8];
  const T* x = (val ? v : k) + tok * (val ? v_st : k_st) + h * (val ? v_sh : k_sh);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[b][e] = 0.f;
    if (slot >= 0) load_quarter<FMT>(x + b * 32, l, f[b]);
  }
  uint32_t w[KW];
  uint16_t d[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    if constexpr (FMT == 0) {
      w[b] = quant_q4_0_quarter(f[b], l, &d[b]);
    } else {
      const uint2 q = quant_q8_0_quarter(f[b], &d[b]);
      w[2 * b] = q.x, w[2 * b + 1] = q.y;
    }
  }
  if (slot < 0) return;
  const int64_t row = (((slot >> page_shift) * c.heads + h) << page_shift) + (slot & ((1 << page_shift) - 1));
  uint8_t* dst = (val ? c.vq : c.kq) + row * kRow + l * (KW * 4);
  if (!val) {
    store_halves<2 * KW>(dst, w);
  } else if constexpr (FMT == 0) {  // the words' low halves are unit 2l, their high halves unit 2l + 1
    uint32_t u[2 * NB + 1];
#pragma unroll
    for (int b = 0; b < NB; ++b) u[b] = w[b] & 0xffffu, u[NB + b] = w[b] >> 16;
    uint32_t y[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) y[b] = u[2 * b] | u[2 * b + 1] << 16;
    store_halves<2 * NB>(dst, y);
  } else {
    uint32_t y[KW];
#pragma unroll
    for (int b = 0; b < NB; ++b) y[b] = w[2 * b], y[NB + b] = w[2 * b + 1];
    store_halves<2 * KW>(dst, y);
  }
  if (l == 0) {
    uint32_t y[(NB + 1) / 2];
#pragma unroll
    for (int b = 0; b < NB; ++b) y[b / 2] = (b & 1) ? (y[b / 2] | (uint32_t)d[b] << 16) : d[b];
    store_halves<NB>(reinterpret_cast<uint8_t*>((val ? c.vs : c.ks) + row * NB), y);
  }
}

template <int FMT, int NB, typename T>
__global__ void __launch_bounds__(256)
    kv_read_kernel(T* __restrict__ k, T* __restrict__ v, const int64_t* __restrict__ slots, b2q_kv_cache c,
                   int page_shift, int64_t ntok) {
  pdl_wait_then_trigger();
  constexpr int kRow = NB * (FMT == 0 ? 16 : 32), KW = kRow / 16;
  const bool val = k == nullptr || blockIdx.y != 0;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x, r = item >> 2;
  const int l = (int)item & 3;
  const int64_t tok = r < (1u << 31) ? (int64_t)((uint32_t)r / (uint32_t)c.heads) : r / c.heads;
  const int h = (int)(r - tok * c.heads);
  if (tok >= ntok) return;
  int64_t slot = slots[tok];
  if (slot >= (c.pages << page_shift)) {
    atomicCAS(&g_kv_error, 0, kErrSlot);
    slot = -1;
  }
  uint32_t w[KW], s[(NB + 1) / 2];
#pragma unroll
  for (int i = 0; i < KW; ++i) w[i] = 0;
#pragma unroll
  for (int i = 0; i < (NB + 1) / 2; ++i) s[i] = 0;
  if (slot >= 0) {
    const int64_t row = (((slot >> page_shift) * c.heads + h) << page_shift) + (slot & ((1 << page_shift) - 1));
    load_halves<2 * KW>((val ? c.vq : c.kq) + row * kRow + l * (KW * 4), w);
    load_halves<NB>(reinterpret_cast<const uint8_t*>((val ? c.vs : c.ks) + row * NB), s);
  }
  if (val) {  // back to [block][word]
    uint32_t y[KW];
#pragma unroll
    for (int i = 0; i < KW; ++i) y[i] = w[i];
    if constexpr (FMT == 0) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const uint32_t lo = (y[b / 2] >> (16 * (b & 1))) & 0xffffu;
        const uint32_t hi = (y[(NB + b) / 2] >> (16 * ((NB + b) & 1))) & 0xffffu;
        w[b] = lo | hi << 16;
      }
    } else {
#pragma unroll
      for (int b = 0; b < NB; ++b) w[2 * b] = y[b], w[2 * b + 1] = y[NB + b];
    }
  }
  T* dst = (val ? v : k) + r * (NB * 32);
  constexpr int kSecond = FMT == 0 ? 16 : 4, kStep = FMT == 0 ? 4 : 8;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const float d = slot >= 0 ? f16_bits_to_f32((uint16_t)(s[b / 2] >> (16 * (b & 1)))) : 0.f;
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (FMT == 0)
        f[e] = d * (float)((int)((w[b] >> ((e & 3) * 8 + (e >> 2) * 4)) & 15) - 8);
      else
        f[e] = d * (float)((int)((w[2 * b + (e >> 2)] >> ((e & 3) * 8)) & 255) - 128);
    }
    if (slot < 0) {  // zeros, not minus zeros
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = 0.f;
    }
    store4(dst + 32 * b + kStep * l, f[0], f[1], f[2], f[3]);
    store4(dst + 32 * b + kStep * l + kSecond, f[4], f[5], f[6], f[7]);
  }
}

int check_kv_cache(const char* who, const b2q_kv_cache* c) {
  if (!c) return fail(B2Q_EINVAL, "%s: null cache", who);
  if (c->fmt != B2Q_FMT_Q4_0 && c->fmt != B2Q_FMT_Q8_0)
    return fail(B2Q_EINVAL, "%s: cache format %d is neither Q4_0 nor Q8_0", who, c->fmt);
  if (c->dim != 64 && c->dim != 96 && c->dim != 128 && c->dim != 256)
    return fail(B2Q_EINVAL, "%s: head dimension %d is not 64, 96, 128 or 256", who, c->dim);
  if (c->heads < 1 || c->heads > 4096) return fail(B2Q_EINVAL, "%s: %d heads (1..4096)", who, c->heads);
  if (c->page < 16 || c->page > 65536 || (c->page & (c->page - 1)))
    return fail(B2Q_EINVAL, "%s: page of %d tokens is not a power of two from 16 to 65536", who, c->page);
  if (c->pages < 0 || c->pages > (int64_t)1 << 31)
    return fail(B2Q_EINVAL, "%s: %lld pages", who, (long long)c->pages);
  if (c->pages && (!c->kq || !c->ks || !c->vq || !c->vs)) return fail(B2Q_EINVAL, "%s: null cache plane", who);
  if (!aligned(c->kq, 16) || !aligned(c->ks, 16) || !aligned(c->vq, 16) || !aligned(c->vs, 16))
    return fail(B2Q_EALIGN, "%s: the cache's planes must be 16-byte aligned", who);
  return B2Q_OK;
}

static int log2_of(int x) {
  int s = 0;
  while ((1 << s) < x) ++s;
  return s;
}

template <int FMT, int NB, typename T>
static int write_as(const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh,
                    const int64_t* slots, const b2q_kv_cache& c, int64_t ntok, cudaStream_t stream) {
  const dim3 grid((unsigned)((ntok * c.heads * 4 + 255) / 256), 2);
  launch_maybe_pdl(kv_write_kernel<FMT, NB, T>, grid, dim3(256), 0, stream, static_cast<const T*>(k), k_st, k_sh,
                   static_cast<const T*>(v), v_st, v_sh, slots, c, log2_of(c.page), ntok);
  return after_launch("kv_write");
}

template <int FMT, int NB, typename T>
static int read_as(void* k, void* v, const int64_t* slots, const b2q_kv_cache& c, int64_t ntok, cudaStream_t stream) {
  const dim3 grid((unsigned)((ntok * c.heads * 4 + 255) / 256), k && v ? 2 : 1);
  launch_maybe_pdl(kv_read_kernel<FMT, NB, T>, grid, dim3(256), 0, stream, static_cast<T*>(k), static_cast<T*>(v),
                   slots, c, log2_of(c.page), ntok);
  return after_launch("kv_read");
}

// Calls fn(format tag, block-count tag, a value of the element type) for the cache's format, dimension and the dtype.
template <int V>
using Tag = std::integral_constant<int, V>;

template <typename Fmt, typename T, typename Fn>
static int by_dim(const b2q_kv_cache& c, Fmt fmt, T elt, Fn fn) {
  switch (c.dim) {
    case 64: return fn(fmt, Tag<2>{}, elt);
    case 96: return fn(fmt, Tag<3>{}, elt);
    case 128: return fn(fmt, Tag<4>{}, elt);
    default: return fn(fmt, Tag<8>{}, elt);
  }
}

template <typename T, typename Fn>
static int by_fmt(const b2q_kv_cache& c, T elt, Fn fn) {
  return c.fmt == B2Q_FMT_Q4_0 ? by_dim(c, Tag<0>{}, elt, fn) : by_dim(c, Tag<2>{}, elt, fn);
}

template <typename Fn>
static int by_type(const b2q_kv_cache& c, int dtype, Fn fn) {
  if (dtype == B2Q_DTYPE_F32) return by_fmt(c, float{}, fn);
  if (dtype == B2Q_DTYPE_F16) return by_fmt(c, __half{}, fn);
  return by_fmt(c, __nv_bfloat16{}, fn);
}

int kv_cache_error(int* code, int clear) { return read_error_word(g_kv_error, code, clear); }

}  // namespace b2q

using namespace b2q;

extern "C" {

int b2q_kv_write(const b2q_kv_cache* cache, int dtype, const void* k, int64_t k_st, int64_t k_sh, const void* v,
                 int64_t v_st, int64_t v_sh, const int64_t* slots, int64_t T, b2q_stream_t stream) {
  const char* who = "b2q_kv_write";
  int rc = check_kv_cache(who, cache);
  if (rc) return rc;
  if (dtype < 0 || dtype > 2) return fail(B2Q_EINVAL, "%s: dtype %d", who, dtype);
  if (T < 0) return fail(B2Q_EINVAL, "%s: T=%lld", who, (long long)T);
  if (T == 0) return B2Q_OK;
  if (!k || !v || !slots) return fail(B2Q_EINVAL, "%s: null pointer", who);
  const int64_t mult = 16 / dtype_size(dtype);
  if (!aligned(k, 16) || !aligned(v, 16) || k_st % mult || k_sh % mult || v_st % mult || v_sh % mult)
    return fail(B2Q_EALIGN, "%s: k and v must be 16-byte aligned, in their strides too", who);
  if (!aligned(slots, 8)) return fail(B2Q_EALIGN, "%s: slots must be 8-byte aligned", who);
  if (T > ((int64_t)1 << 36) / cache->heads) return fail(B2Q_ERANGE, "%s: T=%lld", who, (long long)T);
  return by_type(*cache, dtype, [&](auto fmt, auto nb, auto elt) {
    return write_as<decltype(fmt)::value, decltype(nb)::value, decltype(elt)>(
        k, k_st, k_sh, v, v_st, v_sh, slots, *cache, T, (cudaStream_t)stream);
  });
}

int b2q_kv_read(const b2q_kv_cache* cache, int dtype, void* k, void* v, const int64_t* slots, int64_t T,
                b2q_stream_t stream) {
  const char* who = "b2q_kv_read";
  int rc = check_kv_cache(who, cache);
  if (rc) return rc;
  if (dtype < 0 || dtype > 2) return fail(B2Q_EINVAL, "%s: dtype %d", who, dtype);
  if (T < 0) return fail(B2Q_EINVAL, "%s: T=%lld", who, (long long)T);
  if (T == 0 || (!k && !v)) return B2Q_OK;
  if (!slots) return fail(B2Q_EINVAL, "%s: null pointer", who);
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(slots, 8))
    return fail(B2Q_EALIGN, "%s: k and v must be 16-byte aligned, slots 8-byte aligned", who);
  if (T > ((int64_t)1 << 36) / cache->heads) return fail(B2Q_ERANGE, "%s: T=%lld", who, (long long)T);
  return by_type(*cache, dtype, [&](auto fmt, auto nb, auto elt) {
    return read_as<decltype(fmt)::value, decltype(nb)::value, decltype(elt)>(k, v, slots, *cache, T, (cudaStream_t)stream);
  });
}

}  // extern "C"
