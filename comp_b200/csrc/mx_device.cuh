// Device helpers of the MXFP4 kernels: where a block lies in an operand image, and the 4-bit conversions.
//
// The image is laid out for the tensor cores, so that a kernel brings a stage of a tile (128 rows by 256 values) into shared
// memory with one bulk copy and multiplies it as it lies there:
//   codes   row r is 128 bytes: 8 blocks of 16, block b at place b ^ (r & 7) (the 128-byte swizzle, repeated every 8 rows);
//           in a block byte i holds value i (low nibble) and value i + 16 (high). Both operands have this order, so that
//           their products pair up as they should.
//   scales  after the codes, two runs of 512 bytes (blocks 0..3 and 4..7): byte (r % 32) * 16 + (r / 32) * 4 + b % 4, the
//           order in which tensor memory holds them: lane r % 32, column r / 32.
// Codes and scales of values beyond K are zeros.
#pragma once

#include "kv_device.cuh"
#include "mx_internal.h"

namespace b2q {

// Byte offsets of block b (0..7) of row r (0..127) in a stage: its 16 bytes of codes, its scale.
__device__ __forceinline__ int mx_code_at(int r, int b) { return r * 128 + ((b ^ (r & 7)) << 4); }
__device__ __forceinline__ int mx_scale_at(int r, int b) {
  return kMxCodes + (b >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (b & 3);
}

// 4 bytes of codes, byte i = lo[i] in the low nibble and hi[i] in the high one: round to nearest even, cut off at 6.
__device__ __forceinline__ uint32_t to_e2m1x8(const float (&lo)[8], const float (&hi)[8], int i) {
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %5, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %6, %2;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %7, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %4;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w)
      : "f"(lo[i]), "f"(lo[i + 1]), "f"(lo[i + 2]), "f"(lo[i + 3]), "f"(hi[i]), "f"(hi[i + 1]), "f"(hi[i + 2]),
        "f"(hi[i + 3]));
  return w;
}

// The values of 4 bytes of codes: lo[i] from the low nibble of byte i, hi[i] from the high one.
__device__ __forceinline__ void from_e2m1x8(uint32_t w, float (&lo)[8], float (&hi)[8], int i) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
    lo[i + j] = f.x, hi[i + j] = f.y;
  }
}

// the 8 values from `p` on as f32, and the largest magnitude's bits (a NaN's are above infinity's)
__device__ __forceinline__ uint32_t load8(const float* p, float (&v)[8]) {
  load4(p, *reinterpret_cast<float(*)[4]>(&v[0]));
  load4(p + 4, *reinterpret_cast<float(*)[4]>(&v[4]));
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}
__device__ __forceinline__ uint32_t load8(const __half* p, float (&v)[8]) {
  const uint4 x = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
    m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  }
  m = max(m & 0xffffu, m >> 16);
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
}
__device__ __forceinline__ uint32_t load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 x = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  }
  return max(m << 16, m & 0xffff0000u);
}

// 32 bytes at once (the address a multiple of 32): twice the widest load of older GPUs.
__device__ __forceinline__ void load32(const void* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}

// The scale of a block whose largest magnitude has the bits m (infinities and NaN at the top).
__device__ __forceinline__ uint32_t mx_scale_of(uint32_t m) { return m >= 0x7f800000u ? 255u : max((int)(m >> 23) - 2, 0); }

// Half a block, values 8h .. 8h + 7 and 16 + 8h .. 16 + 8h + 7 from `p` on (the two nibbles of bytes 8h .. 8h + 7), by one of two
// neighbouring lanes; finish() gives the block's scale and leaves the codes. All 32 lanes call it.
struct MxHalf {
  float lo[8], hi[8];
  uint32_t largest = 0;
  uint2 codes;

  template <typename T>
  __device__ __forceinline__ void load(const T* p, bool there) {
    if (there) {
      largest = load8(p, lo);
      largest = max(largest, load8(p + 16, hi));
    } else {
      clear();
    }
  }
  __device__ __forceinline__ void clear() {
    largest = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = hi[i] = 0.f;
  }
  // (s: the scale; codes of a block that is NaN are zeros)
  __device__ __forceinline__ void encode(uint32_t s) {
    const float up = __uint_as_float((254 - s) << 23);  // 2^(127 - s)
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] *= up, hi[i] *= up;
    codes = s == 255 ? make_uint2(0, 0) : make_uint2(to_e2m1x8(lo, hi, 0), to_e2m1x8(lo, hi, 4));
  }
  __device__ __forceinline__ uint32_t finish() {
    const uint32_t s = mx_scale_of(max(largest, __shfl_xor_sync(0xffffffffu, largest, 1)));
    encode(s);
    return s;
  }
};

// 2^(s - 127): s = 0 is below the normal numbers, 255 is NaN.
__device__ __forceinline__ float mx_scale(uint32_t s) {
  return __uint_as_float(s == 0 ? 0x00400000u : s == 255 ? 0x7fffffffu : s << 23);
}

}  // namespace b2q
