// MXFP4 on the tensor cores: descriptors, scale copies and products of operands that lie in shared memory as in their images
// (PTX ISA 8.7, sm_100a).
#pragma once

#include "mx_device.cuh"
#include "tc_device.cuh"

namespace b2q {

// One lane of a converged warp, told in the way that lets the compiler see that it is one: tensor-core instructions take
// their operands from uniform registers, and behind a branch on the lane's number each issues some four times as slowly (a stage's
// six scale copies and four products 900 cycles, so 220).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

// K-major operand with the 128-byte swizzle: 8 rows every 1024 bytes
__device__ __forceinline__ uint64_t desc_swizzled(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// 32 rows of 16 bytes without swizzle: 8 rows every 128 bytes
__device__ __forceinline__ uint64_t desc_scales(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
}
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t smem) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc_scales(smem)) : "memory");
}
// kind::mxf4: f32 accumulator, A and B e2m1, both K-major, M = 128, N = n, ue8m0 scales; `half`: which two of a column's four
// scale bytes count
__device__ __forceinline__ uint32_t instr_desc_mxf4(int n, int half) {
  const uint32_t id = half ? 2u : 0u;
  return (id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | (8u << 24) | (id << 29);
}
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                         uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void store_one(float* y, float v) { *y = v; }
__device__ __forceinline__ void store_one(__half* y, float v) { *y = __float2half_rn(v); }
__device__ __forceinline__ void store_one(__nv_bfloat16* y, float v) { *y = __float2bfloat16_rn(v); }
// f(y as its type): the type is looked at once for all that f stores
template <typename F>
__device__ __forceinline__ void with_type(void* y, int dtype, F f) {
  if (dtype == B2Q_DTYPE_BF16) f(static_cast<__nv_bfloat16*>(y));
  else if (dtype == B2Q_DTYPE_F16) f(static_cast<__half*>(y));
  else f(static_cast<float*>(y));
}
__device__ __forceinline__ void store_as(void* y, int64_t at, int dtype, float v) {
  if (dtype == B2Q_DTYPE_BF16)
    static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
  else if (dtype == B2Q_DTYPE_F16)
    static_cast<__half*>(y)[at] = __float2half_rn(v);
  else
    static_cast<float*>(y)[at] = v;
}

}  // namespace b2q
