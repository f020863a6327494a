// Quantized KV cache: quantizing keys and values into their slots, and reading slots back.
//
// Both are one pass, bound by memory: a write reads the values once and stores 4.5 (q4_0) or 8.5 (q8_0) bits for each,
// a read the reverse. A thread takes a quarter of a 32-value block (8 values): for q4_0 the values 4l..4l+3 and
// 16+4l..16+4l+3, which are the two nibbles of the block's bytes 4l..4l+3 (one key unit, two value units), for q8_0 the
// values 8l..8l+7. Every 32-byte sector of input, quants and output is then touched by one warp in whole.
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

// ggml's q4_0 block of 32 values held by 4 consecutive lanes (values 4l.. and 16+4l..): the lane's 4 bytes, f16 d bits.
__device__ __forceinline__ uint32_t quant_q4_0_quarter(const float (&v)[8], int l, uint16_t* d_bits) {
  float best = 0.f, mag = -1.f;
  int at = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(v[i]);
    const int idx = (i < 4 ? 0 : 12) + 4 * l + i;
    if (a > mag) mag = a, best = v[i], at = idx;  // ascending: the first of equals stays
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, mag, o), b2 = __shfl_xor_sync(0xffffffffu, best, o);
    const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
    if (m2 > mag || (m2 == mag && a2 < at)) mag = m2, best = b2, at = a2;
  }
  const float d = __fmul_rn(best, -0.125f);  // m / -8, exact but for underflow
  const float id = d != 0.f ? __fdiv_rn(1.0f, d) : 0.f;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int q = max(0, min(15, (int)__fadd_rn(__fmul_rn(v[i], id), 8.5f)));
    w |= (uint32_t)q << ((i & 3) * 8 + (i >> 2) * 4);
  }
  *d_bits = __half_as_ushort(__float2half_rn(d));
  return w;
}

// ggml's q8_0 block, the quants plus 128: the lane's 8 bytes (values 8l..8l+7).
__device__ __forceinline__ uint2 quant_q8_0_quarter(const float (&v)[8], uint16_t* d_bits) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  const float d = __fdiv_rn(amax, 127.0f);
  const float id = d != 0.f ? __fdiv_rn(1.0f, d) : 0.f;
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int q = (int)roundf(__fmul_rn(v[i], id)) + 128;
    w[i >> 2] |= (uint32_t)(q & 0xff) << ((i & 3) * 8);
  }
  *d_bits = __half_as_ushort(__float2half_rn(d));
  return make_uint2(w[0], w[1]);
}

// One thread per (token, head, block, quarter); blockIdx.y 0 = keys, 1 = values. `tpb` tokens a CTA.
template <int FMT, int NB, typename T>
__global__ void __launch_bounds__(256)
    kv_write_kernel(const T* __restrict__ k, int64_t k_st, int64_t k_sh, const T* __restrict__ v, int64_t v_st,
                    int64_t v_sh, const int64_t* __restrict__ slots, b2q_kv_cache c, int page_shift, int64_t ntok,
                    int tpb) {
  pdl_wait_then_trigger();
  constexpr int kRow = NB * (FMT == 0 ? 16 : 32);
  const bool val = blockIdx.y != 0;
  const T* x = val ? v : k;
  const int64_t st = val ? v_st : k_st, sh = val ? v_sh : k_sh;
  uint8_t* quants = val ? c.vq : c.kq;
  int16_t* scales = val ? c.vs : c.ks;
  const int per_token = c.heads * NB * 4;
  const int items = tpb * per_token;
  const int64_t t0 = (int64_t)blockIdx.x * tpb;
  for (int base = 0; base < items; base += 256) {  // CTA-uniform: the shuffles need whole warps
    const int i = base + threadIdx.x;
    const int tt = i / per_token, r = i - tt * per_token;
    const int64_t tok = t0 + tt;
    const int l = r & 3, b = (r >> 2) % NB, h = (r >> 2) / NB;
    int64_t slot = -1;
    if (i < items && tok < ntok) slot = slots[tok];
    if (slot >= (c.pages << page_shift)) {
      atomicCAS(&g_kv_error, 0, kErrSlot);
      slot = -1;
    }
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (slot >= 0) load_quarter<FMT>(x + tok * st + h * sh + b * 32, l, f);
    uint16_t d;
    const int64_t row = ((slot >> page_shift) * c.heads + h << page_shift) + (slot & ((1 << page_shift) - 1));
    if constexpr (FMT == 0) {
      const uint32_t w = quant_q4_0_quarter(f, l, &d);
      if (slot >= 0) {
        uint8_t* dst = quants + row * kRow;
        if (!val) {
          *reinterpret_cast<uint32_t*>(dst + (l * NB + b) * 4) = w;
        } else {
          *reinterpret_cast<uint16_t*>(dst + ((2 * l) * NB + b) * 2) = (uint16_t)w;
          *reinterpret_cast<uint16_t*>(dst + ((2 * l + 1) * NB + b) * 2) = (uint16_t)(w >> 16);
        }
      }
    } else {
      const uint2 w = quant_q8_0_quarter(f, &d);
      if (slot >= 0) {
        uint8_t* dst = quants + row * kRow;
        if (!val) {
          *reinterpret_cast<uint2*>(dst + (l * NB + b) * 8) = w;
        } else {
          *reinterpret_cast<uint32_t*>(dst + ((2 * l) * NB + b) * 4) = w.x;
          *reinterpret_cast<uint32_t*>(dst + ((2 * l + 1) * NB + b) * 4) = w.y;
        }
      }
    }
    if (slot >= 0 && l == 0) scales[row * NB + b] = (int16_t)d;
  }
}

template <int FMT, int NB, typename T>
__global__ void __launch_bounds__(256)
    kv_read_kernel(T* __restrict__ k, T* __restrict__ v, const int64_t* __restrict__ slots, b2q_kv_cache c,
                   int page_shift, int64_t ntok, int tpb) {
  pdl_wait_then_trigger();
  constexpr int kRow = NB * (FMT == 0 ? 16 : 32);
  const bool val = k == nullptr || blockIdx.y != 0;
  T* x = val ? v : k;
  const uint8_t* quants = val ? c.vq : c.kq;
  const int16_t* scales = val ? c.vs : c.ks;
  const int per_token = c.heads * NB * 4;
  const int items = tpb * per_token;
  const int64_t t0 = (int64_t)blockIdx.x * tpb;
  for (int i = threadIdx.x; i < items; i += 256) {
    const int tt = i / per_token, r = i - tt * per_token;
    const int64_t tok = t0 + tt;
    if (tok >= ntok) return;
    const int l = r & 3, b = (r >> 2) % NB, h = (r >> 2) / NB;
    int64_t slot = slots[tok];
    if (slot >= (c.pages << page_shift)) {
      atomicCAS(&g_kv_error, 0, kErrSlot);
      slot = -1;
    }
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (slot >= 0) {
      const int64_t row = ((slot >> page_shift) * c.heads + h << page_shift) + (slot & ((1 << page_shift) - 1));
      const float d = f16_bits_to_f32((uint16_t)scales[row * NB + b]);
      const uint8_t* src = quants + row * kRow;
      if constexpr (FMT == 0) {
        uint32_t w;
        if (!val)
          w = *reinterpret_cast<const uint32_t*>(src + (l * NB + b) * 4);
        else
          w = *reinterpret_cast<const uint16_t*>(src + ((2 * l) * NB + b) * 2) |
              (uint32_t) * reinterpret_cast<const uint16_t*>(src + ((2 * l + 1) * NB + b) * 2) << 16;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = d * (float)((int)((w >> ((e & 3) * 8 + (e >> 2) * 4)) & 15) - 8);
      } else {
        uint2 w;
        if (!val) {
          w = *reinterpret_cast<const uint2*>(src + (l * NB + b) * 8);
        } else {
          w.x = *reinterpret_cast<const uint32_t*>(src + ((2 * l) * NB + b) * 4);
          w.y = *reinterpret_cast<const uint32_t*>(src + ((2 * l + 1) * NB + b) * 4);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
          f[e] = d * (float)((int)(((e < 4 ? w.x : w.y) >> ((e & 3) * 8)) & 255) - 128);
      }
    }
    T* dst = x + (tok * c.heads + h) * (NB * 32) + b * 32;
    constexpr int kSecond = FMT == 0 ? 16 : 4, kStep = FMT == 0 ? 4 : 8;
    store4(dst + kStep * l, f[0], f[1], f[2], f[3]);
    store4(dst + kStep * l + kSecond, f[4], f[5], f[6], f[7]);
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

// Tokens a CTA: about 1024 threads' items, fewer when the tokens alone do not fill the GPU.
static int tokens_per_cta(int64_t T, int per_token) {
  DeviceInfo di;
  const int sms = device_info(&di) == B2Q_OK ? di.sms : 148;
  int tpb = 1024 / per_token;
  if (tpb > T / (2 * sms)) tpb = (int)(T / (2 * sms));
  return tpb < 1 ? 1 : tpb;
}

template <int FMT, int NB, typename T>
static int write_as(const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh,
                    const int64_t* slots, const b2q_kv_cache& c, int64_t ntok, cudaStream_t stream) {
  const int tpb = tokens_per_cta(ntok, c.heads * NB * 4);
  const dim3 grid((unsigned)((ntok + tpb - 1) / tpb), 2);
  launch_maybe_pdl(kv_write_kernel<FMT, NB, T>, grid, dim3(256), 0, stream, static_cast<const T*>(k), k_st, k_sh,
                   static_cast<const T*>(v), v_st, v_sh, slots, c, log2_of(c.page), ntok, tpb);
  return after_launch("kv_write");
}

template <int FMT, int NB, typename T>
static int read_as(void* k, void* v, const int64_t* slots, const b2q_kv_cache& c, int64_t ntok, cudaStream_t stream) {
  const int tpb = tokens_per_cta(ntok, c.heads * NB * 4);
  const dim3 grid((unsigned)((ntok + tpb - 1) / tpb), k && v ? 2 : 1);
  launch_maybe_pdl(kv_read_kernel<FMT, NB, T>, grid, dim3(256), 0, stream, static_cast<T*>(k), static_cast<T*>(v),
                   slots, c, log2_of(c.page), ntok, tpb);
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
  if (T > (int64_t)1 << 31) return fail(B2Q_ERANGE, "%s: T=%lld", who, (long long)T);
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
  if (T > (int64_t)1 << 31) return fail(B2Q_ERANGE, "%s: T=%lld", who, (long long)T);
  return by_type(*cache, dtype, [&](auto fmt, auto nb, auto elt) {
    return read_as<decltype(fmt)::value, decltype(nb)::value, decltype(elt)>(k, v, slots, *cache, T, (cudaStream_t)stream);
  });
}

}  // extern "C"
