// MXFP4 operand images: quantized from rows of values, packed from planes of codes and scales, read back as values.
//
// A block of 32 values has the scale 2^(s - 127), s = max(0, floor(log2 max|x|) + 125): the exponent of the largest
// magnitude less 2, so that this lies in 4 .. 8 of the 4-bit values' range (largest: 6, larger ones are cut off). A value times
// the scale's inverse, a power of two, is exact; the conversion rounds it once, to nearest even. A block with an infinity
// or a NaN has s = 255, NaN.
//
// All three are one pass, bound by memory: a thread a block, values in runs of 32 bytes (a sector) where the rows are
// aligned to them, else of 16, and 16 bytes of codes. 16384 x 8192 bf16 values: 56 us (6.0 TB/s), and read back 109 in all; two
// threads a block, with 16-byte loads, took 122. Planes of 8192 x 8192 packed: 13 us (5.5 TB/s), of 32 x 4096 x 4096 100 us (5.7).
#include <type_traits>

#include "mx_device.cuh"

namespace b2q {

int check_mx_shape(const char* who, int64_t rows, int64_t K) {
  if (rows < 0 || rows > INT32_MAX - 1024) return fail(B2Q_EINVAL, "%s: %lld rows", who, (long long)rows);
  if (K < 32 || K % 32 || K > INT32_MAX / 2)
    return fail(B2Q_EINVAL, "%s: K=%lld is not a positive multiple of 32", who, (long long)K);
  return B2Q_OK;
}

int check_mx_rows(const char* who, const char* name, int dtype, const void* x, int64_t ldx, int64_t rows, int64_t K) {
  if (dtype < B2Q_DTYPE_F32 || dtype > B2Q_DTYPE_BF16) return fail(B2Q_EINVAL, "%s: %s: unknown dtype %d", who, name, dtype);
  if (rows == 0) return B2Q_OK;
  if (!x) return fail(B2Q_EINVAL, "%s: %s is NULL", who, name);
  if (ldx < K && rows > 1) return fail(B2Q_EINVAL, "%s: %s: row stride %lld < %lld", who, name, (long long)ldx, (long long)K);
  return B2Q_OK;
}

namespace {

// 16 values from `p` on as f32, and their largest magnitude's bits. WIDE: the address is a multiple of 32 bytes.
template <bool WIDE, typename T>
__device__ __forceinline__ uint32_t load16(const T* p, float (&a)[8], float (&b)[8]) {
  if constexpr (!WIDE) return max(load8(p, a), load8(p + 8, b));
  uint32_t w[8], m = 0;
  load32(p, w);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = __uint_as_float(w[i]), m = max(m, w[i] & 0x7fffffffu);
    load32(p + 8, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = __uint_as_float(w[i]), m = max(m, w[i] & 0x7fffffffu);
    return m;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float* v = (i < 4 ? a : b) + 2 * (i & 3);
      if constexpr (std::is_same_v<T, __half>) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[0] = f.x, v[1] = f.y;
      } else {
        v[0] = __uint_as_float(w[i] << 16), v[1] = __uint_as_float(w[i] & 0xffff0000u);
      }
      m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    }
    if constexpr (std::is_same_v<T, __half>)
      return __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(m & 0xffffu, m >> 16))));
    else
      return max(m << 16, m & 0xffff0000u);
  }
}

// 16 values to `p`.
template <bool WIDE, typename T>
__device__ __forceinline__ void store16(T* p, const float (&a)[8], const float (&b)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float(&v)[8] = h ? b : a;
      if constexpr (WIDE)
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p + 8 * h), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                     "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                     : "memory");
      else
        store4(p + 8 * h, v[0], v[1], v[2], v[3]), store4(p + 8 * h + 4, v[4], v[5], v[6], v[7]);
    }
  } else {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = (i < 4 ? a : b)[2 * (i & 3)], y = (i < 4 ? a : b)[2 * (i & 3) + 1];
      if constexpr (std::is_same_v<T, __half>) {
        w[i] = pack_half2(x, y);
      } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
    if constexpr (WIDE) {
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                   "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                   : "memory");
    } else {
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(p + 8) = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
}

// A thread's place: block b of a stage of a row; 8 threads a stage.
struct Place {
  int64_t row;
  int stage, b;
};
__device__ __forceinline__ Place place_of(int64_t item, int stages) {
  const int64_t s = item >> 3;
  const int64_t row = s < (1ll << 31) ? (int64_t)((uint32_t)s / (uint32_t)stages) : s / stages;
  return {row, (int)(s - row * stages), (int)item & 7};
}

// The image's row of row r of operands of `each` rows, which begin at whole tiles.
__device__ __forceinline__ int64_t image_row(int64_t r, int64_t each) {
  if (r < each) return r;
  const int64_t e = r / each;
  return e * ((each + kMxRows - 1) / kMxRows * kMxRows) + (r - e * each);
}

template <bool WIDE, typename T>
__global__ void __launch_bounds__(256)
    mx_quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int64_t each, int K, int stages,
                       uint8_t* __restrict__ image, const int32_t* __restrict__ dest, int fan) {
  pdl_wait_then_trigger();
  const Place p = place_of((int64_t)blockIdx.x * 256 + threadIdx.x, stages);
  const int at = p.stage * kMxStage + p.b * 32;
  uint32_t m = 0;
  MxHalf h[2] = {};
  if (p.row < rows && at < K) {  // K is a multiple of 32: a whole block is there, or none of it
    const T* src = x + p.row * ldx + at;
    m = load16<WIDE>(src, h[0].lo, h[1].lo);
    m = max(m, load16<WIDE>(src + 16, h[0].hi, h[1].hi));
  }
  const uint32_t s = mx_scale_of(m);
  h[0].encode(s), h[1].encode(s);
  uint32_t scales = s << (8 * (p.b & 3));  // the 4 blocks of a word: 4 lanes of the same row
  scales |= __shfl_xor_sync(0xffffffffu, scales, 1);
  scales |= __shfl_xor_sync(0xffffffffu, scales, 2);
  if (p.row >= rows) return;
  const int64_t first = dest ? p.row * fan : 0;
  for (int j = 0; j < fan; ++j) {
    const int64_t r = dest ? dest[first + j] : image_row(p.row, each);
    if (r < 0) continue;
    uint8_t* tile = image + ((r >> 7) * stages + p.stage) * kMxBytes;
    const int in = (int)r & 127;
    *reinterpret_cast<uint4*>(tile + mx_code_at(in, p.b)) = make_uint4(h[0].codes.x, h[0].codes.y, h[1].codes.x, h[1].codes.y);
    if ((p.b & 3) == 0) *reinterpret_cast<uint32_t*>(tile + mx_scale_at(in, p.b)) = scales;
  }
}

template <bool WIDE, typename T>
__global__ void __launch_bounds__(256)
    mx_dequantize_kernel(const uint8_t* __restrict__ image, int64_t rows, int64_t each, int K, int stages, T* __restrict__ y,
                         int64_t ldy) {
  pdl_wait_then_trigger();
  const Place p = place_of((int64_t)blockIdx.x * 256 + threadIdx.x, stages);
  const int at = p.stage * kMxStage + p.b * 32;
  if (p.row >= rows || at >= K) return;
  const int64_t r = image_row(p.row, each);
  const uint8_t* tile = image + ((r >> 7) * stages + p.stage) * kMxBytes;
  const int in = (int)r & 127;
  const uint4 q = *reinterpret_cast<const uint4*>(tile + mx_code_at(in, p.b));
  const float d = mx_scale(tile[mx_scale_at(in, p.b)]);
  float lo[2][8], hi[2][8];
  from_e2m1x8(q.x, lo[0], hi[0], 0);
  from_e2m1x8(q.y, lo[0], hi[0], 4);
  from_e2m1x8(q.z, lo[1], hi[1], 0);
  from_e2m1x8(q.w, lo[1], hi[1], 4);
#pragma unroll
  for (int i = 0; i < 8; ++i) lo[0][i] *= d, hi[0][i] *= d, lo[1][i] *= d, hi[1][i] *= d;
  T* dst = y + p.row * ldy + at;
  store16<WIDE>(dst, lo[0], lo[1]);
  store16<WIDE>(dst + 16, hi[0], hi[1]);
}

// Planes [experts][rows] of codes and scales into an image whose experts begin at whole tiles; rows beyond the last are zeros.
__global__ void __launch_bounds__(256)
    mx_pack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int experts, int rows, int row_tiles,
                   int K, int stages, uint8_t* __restrict__ image) {
  pdl_wait_then_trigger();
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;  // a block of 32 values each
  const int64_t s = item >> 3, row = s / stages;
  const int stage = (int)(s - row * stages), b = (int)item & 7, block = stage * 8 + b;
  const int64_t tile = row >> 7, e = tile / row_tiles;
  if (e >= experts) return;
  const int in = (int)row & 127;
  const int64_t r = (tile - e * row_tiles) * 128 + in;
  uint4 q = {0, 0, 0, 0};
  uint8_t d = 0;
  if (r < rows && block < K / 32) {
    const int64_t at = (e * rows + r) * (K / 32) + block;
    q = *reinterpret_cast<const uint4*>(codes + at * 16);
    d = scales[at];
  }
  uint8_t* dst = image + (tile * stages + stage) * kMxBytes;
  *reinterpret_cast<uint4*>(dst + mx_code_at(in, b)) = q;
  dst[mx_scale_at(in, b)] = d;
}

int check_experts(const char* who, int64_t experts, int64_t rows, int64_t K) {
  if (experts < 1 || experts > kMaxExperts)
    return fail(B2Q_EINVAL, "%s: %lld experts (1..%lld)", who, (long long)experts, (long long)kMaxExperts);
  if (experts * mx_tiles(rows) * mx_stages(K) > INT64_MAX / kMxBytes)
    return fail(B2Q_ERANGE, "%s: %lld x %lld x %lld values are past 64-bit sizes", who, (long long)experts, (long long)rows, (long long)K);
  return B2Q_OK;
}

int grid_of(const char* who, int64_t items, unsigned* grid) {
  const int64_t n = (items + 255) / 256;
  if (n > INT32_MAX) return fail(B2Q_ERANGE, "%s: too many values for one launch", who);
  *grid = (unsigned)n;
  return B2Q_OK;
}

}  // namespace

int launch_mx_quantize(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t each, int64_t K, uint8_t* image,
                       const int32_t* dest, int fan, cudaStream_t stream) {
  const int stages = (int)mx_stages(K);
  unsigned grid;
  int rc = grid_of("b2q_mx_quantize", rows * stages * 8, &grid);
  if (rc || rows == 0) return rc;
  const bool wide = aligned(x, 32) && (rows == 1 || ldx * mx_dtype_size(dtype) % 32 == 0);
  auto launch = [&](auto kernel, auto* p) {
    launch_maybe_pdl(kernel, dim3(grid), dim3(256), 0, stream, p, ldx, rows, each, (int)K, stages, image, dest, fan);
  };
  if (dtype == B2Q_DTYPE_F32)
    launch(wide ? mx_quantize_kernel<true, float> : mx_quantize_kernel<false, float>, static_cast<const float*>(x));
  else if (dtype == B2Q_DTYPE_F16)
    launch(wide ? mx_quantize_kernel<true, __half> : mx_quantize_kernel<false, __half>, static_cast<const __half*>(x));
  else
    launch(wide ? mx_quantize_kernel<true, __nv_bfloat16> : mx_quantize_kernel<false, __nv_bfloat16>,
           static_cast<const __nv_bfloat16*>(x));
  return after_launch("mx_quantize");
}

}  // namespace b2q

using namespace b2q;

extern "C" {

size_t b2q_mx_bytes(int64_t experts, int64_t rows, int64_t K) {
  if (check_mx_shape("b2q_mx_bytes", rows, K)) return 0;
  if (check_experts("b2q_mx_bytes", experts, rows, K)) return 0;
  return (size_t)experts * mx_tiles(rows) * mx_stages(K) * kMxBytes;
}

int b2q_mx_quantize(int dtype, const void* x, int64_t ldx, int64_t experts, int64_t rows, int64_t K, uint8_t* image,
                    b2q_stream_t stream) {
  const char* who = "b2q_mx_quantize";
  int rc = check_mx_shape(who, rows, K);
  if (!rc) rc = check_experts(who, experts, rows, K);
  if (!rc) rc = check_mx_rows(who, "x", dtype, x, ldx, experts * rows, K);
  if (rc || rows == 0) return rc;
  if (!image) return fail(B2Q_EINVAL, "%s: image is NULL", who);
  if (!aligned(x, 16) || (experts * rows > 1 && ldx * mx_dtype_size(dtype) % 16) || !aligned(image, 128))
    return fail(B2Q_EALIGN, "%s: x and its row stride must be 16-byte aligned, the image 128-byte", who);
  return launch_mx_quantize(dtype, x, ldx, experts * rows, rows, K, image, nullptr, 1, stream);
}

int b2q_mx_dequantize(const uint8_t* image, int64_t experts, int64_t each, int64_t K, int dtype, void* y, int64_t ldy,
                      b2q_stream_t stream) {
  const char* who = "b2q_mx_dequantize";
  int rc = check_mx_shape(who, each, K);
  if (!rc) rc = check_experts(who, experts, each, K);
  const int64_t rows = rc ? 0 : experts * each;
  if (!rc) rc = check_mx_rows(who, "y", dtype, y, ldy, rows, K);
  if (rc || rows == 0) return rc;
  if (!image) return fail(B2Q_EINVAL, "%s: image is NULL", who);
  if (!aligned(y, 16) || (rows > 1 && ldy * mx_dtype_size(dtype) % 16) || !aligned(image, 128))
    return fail(B2Q_EALIGN, "%s: y and its row stride must be 16-byte aligned, the image 128-byte", who);
  const int stages = (int)mx_stages(K);
  unsigned grid;
  rc = grid_of(who, rows * stages * 8, &grid);
  if (rc) return rc;
  const bool wide = aligned(y, 32) && (rows == 1 || ldy * mx_dtype_size(dtype) % 32 == 0);
  auto launch = [&](auto kernel, auto* p) {
    launch_maybe_pdl(kernel, dim3(grid), dim3(256), 0, stream, image, rows, each, (int)K, stages, p, ldy);
  };
  if (dtype == B2Q_DTYPE_F32)
    launch(wide ? mx_dequantize_kernel<true, float> : mx_dequantize_kernel<false, float>, static_cast<float*>(y));
  else if (dtype == B2Q_DTYPE_F16)
    launch(wide ? mx_dequantize_kernel<true, __half> : mx_dequantize_kernel<false, __half>, static_cast<__half*>(y));
  else
    launch(wide ? mx_dequantize_kernel<true, __nv_bfloat16> : mx_dequantize_kernel<false, __nv_bfloat16>,
           static_cast<__nv_bfloat16*>(y));
  return after_launch("mx_dequantize");
}

int b2q_mx_pack(const uint8_t* codes, const uint8_t* scales, int64_t experts, int64_t rows, int64_t K, uint8_t* image,
                b2q_stream_t stream) {
  const char* who = "b2q_mx_pack";
  int rc = check_mx_shape(who, rows, K);
  if (!rc) rc = check_experts(who, experts, rows, K);
  if (rc || rows == 0) return rc;
  if (!codes || !scales || !image) return fail(B2Q_EINVAL, "%s: null pointer", who);
  if (!aligned(codes, 16) || !aligned(image, 128))
    return fail(B2Q_EALIGN, "%s: codes must be 16-byte aligned, the image 128-byte", who);
  const int64_t tiles = mx_tiles(rows), stages = mx_stages(K);
  unsigned grid;
  rc = grid_of(who, experts * tiles * kMxRows * stages * 8, &grid);
  if (rc) return rc;
  launch_maybe_pdl(mx_pack_kernel, grid, 256, 0, stream, codes, scales, (int)experts, (int)rows, (int)tiles, (int)K, (int)stages,
                   image);
  return after_launch("mx_pack");
}

}  // extern "C"
