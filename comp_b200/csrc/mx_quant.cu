// MXFP4 operand images: quantized from rows of values, packed from planes of codes and scales, read back as values.
//
// A block of 32 values has the scale 2^(s - 127), s = max(0, floor(log2 max|x|) + 125): the exponent of the largest
// magnitude less 2, so that this lies in 4 .. 8 of the 4-bit values' range (largest: 6, larger ones are cut off). A value times
// the scale's inverse, a power of two, is exact; the conversion rounds it once, to nearest even. A block with an infinity
// or a NaN has s = 255, NaN.
//
// All three are one pass, bound by memory. Two threads take a block, values 8h .. 8h + 7 and 16 + 8h .. 16 + 8h + 7 (the two
// nibbles of bytes 8h .. 8h + 7): 16-byte loads of 16-bit values whose pairs make whole 32-byte sectors, and one 8-byte
// store each.
#include "mx_device.cuh"

namespace b2q {

int check_mx_shape(const char* who, int64_t rows, int64_t K) {
  if (rows < 0 || rows > INT32_MAX) return fail(B2Q_EINVAL, "%s: %lld rows", who, (long long)rows);
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

__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  store4(p, v[0], v[1], v[2], v[3]);
  store4(p + 4, v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__half* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_half2(v[0], v[1]), pack_half2(v[2], v[3]), pack_half2(v[4], v[5]), pack_half2(v[6], v[7]));
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// A thread's place: half block `half` of block b of a stage of a row; 16 threads a stage.
struct Place {
  int64_t row;
  int stage, b, half;
};
__device__ __forceinline__ Place place_of(int64_t item, int stages) {
  const int64_t s = item >> 4;
  const int64_t row = s < (1ll << 31) ? (int64_t)((uint32_t)s / (uint32_t)stages) : s / stages;
  return {row, (int)(s - row * stages), (int)(item >> 1) & 7, (int)item & 1};
}

template <typename T>
__global__ void __launch_bounds__(256)
    mx_quantize_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int K, int stages, uint8_t* __restrict__ image,
                       const int32_t* __restrict__ dest, int fan) {
  pdl_wait_then_trigger();
  const Place p = place_of((int64_t)blockIdx.x * 256 + threadIdx.x, stages);
  const int at = p.stage * kMxStage + p.b * 32 + 8 * p.half;
  const bool there = p.row < rows && at < K;  // K is a multiple of 32: a whole block is there, or none of it
  MxHalf h;
  h.load(x + p.row * ldx + at, there);
  const uint32_t s = h.finish();
  uint32_t scales = s << (8 * (p.b & 3));  // the 4 blocks of a word: 8 lanes of the same row
  scales |= __shfl_xor_sync(0xffffffffu, scales, 2);
  scales |= __shfl_xor_sync(0xffffffffu, scales, 4);
  if (p.row >= rows) return;
  const int64_t first = dest ? p.row * fan : 0;
  for (int j = 0; j < fan; ++j) {
    const int64_t r = dest ? dest[first + j] : p.row;
    if (r < 0) continue;
    uint8_t* tile = image + ((r >> 7) * stages + p.stage) * kMxBytes;
    const int in = (int)r & 127;
    *reinterpret_cast<uint2*>(tile + mx_code_at(in, p.b) + 8 * p.half) = h.codes;
    if ((threadIdx.x & 7) == 0) *reinterpret_cast<uint32_t*>(tile + mx_scale_at(in, p.b)) = scales;
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
    mx_dequantize_kernel(const uint8_t* __restrict__ image, int64_t rows, int K, int stages, T* __restrict__ y, int64_t ldy) {
  pdl_wait_then_trigger();
  const Place p = place_of((int64_t)blockIdx.x * 256 + threadIdx.x, stages);
  const int at = p.stage * kMxStage + p.b * 32 + 8 * p.half;
  if (p.row >= rows || at >= K) return;
  const uint8_t* tile = image + ((p.row >> 7) * stages + p.stage) * kMxBytes;
  const int in = (int)p.row & 127;
  const uint2 q = *reinterpret_cast<const uint2*>(tile + mx_code_at(in, p.b) + 8 * p.half);
  const float d = mx_scale(tile[mx_scale_at(in, p.b)]);
  float lo[8], hi[8];
  from_e2m1x8(q.x, lo, hi, 0);
  from_e2m1x8(q.y, lo, hi, 4);
#pragma unroll
  for (int i = 0; i < 8; ++i) lo[i] *= d, hi[i] *= d;
  T* dst = y + p.row * ldy + at;
  store8(dst, lo);
  store8(dst + 16, hi);
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

int grid_of(const char* who, int64_t items, unsigned* grid) {
  const int64_t n = (items + 255) / 256;
  if (n > INT32_MAX) return fail(B2Q_ERANGE, "%s: too many values for one launch", who);
  *grid = (unsigned)n;
  return B2Q_OK;
}

}  // namespace

int launch_mx_quantize(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t K, uint8_t* image, const int32_t* dest,
                       int fan, cudaStream_t stream) {
  const int stages = (int)mx_stages(K);
  unsigned grid;
  int rc = grid_of("b2q_mx_quantize", rows * stages * 16, &grid);
  if (rc || rows == 0) return rc;
  if (dtype == B2Q_DTYPE_F32)
    launch_maybe_pdl(mx_quantize_kernel<float>, grid, 256, 0, stream, static_cast<const float*>(x), ldx, rows, (int)K, stages,
                     image, dest, fan);
  else if (dtype == B2Q_DTYPE_F16)
    launch_maybe_pdl(mx_quantize_kernel<__half>, grid, 256, 0, stream, static_cast<const __half*>(x), ldx, rows, (int)K, stages,
                     image, dest, fan);
  else
    launch_maybe_pdl(mx_quantize_kernel<__nv_bfloat16>, grid, 256, 0, stream, static_cast<const __nv_bfloat16*>(x), ldx, rows,
                     (int)K, stages, image, dest, fan);
  return after_launch("mx_quantize");
}

}  // namespace b2q

using namespace b2q;

extern "C" {

size_t b2q_mx_bytes(int64_t experts, int64_t rows, int64_t K) {
  if (check_mx_shape("b2q_mx_bytes", rows, K)) return 0;
  if (experts < 1 || experts > kMaxExperts) {
    fail(B2Q_EINVAL, "b2q_mx_bytes: %lld experts (1..%lld)", (long long)experts, (long long)kMaxExperts);
    return 0;
  }
  return (size_t)experts * mx_tiles(rows) * mx_stages(K) * kMxBytes;
}

int b2q_mx_quantize(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t K, uint8_t* image, b2q_stream_t stream) {
  const char* who = "b2q_mx_quantize";
  int rc = check_mx_shape(who, rows, K);
  if (!rc) rc = check_mx_rows(who, "x", dtype, x, ldx, rows, K);
  if (rc || rows == 0) return rc;
  if (!image) return fail(B2Q_EINVAL, "%s: image is NULL", who);
  if (!aligned(x, 16) || (rows > 1 && ldx * mx_dtype_size(dtype) % 16) || !aligned(image, 128))
    return fail(B2Q_EALIGN, "%s: x and its row stride must be 16-byte aligned, the image 128-byte", who);
  return launch_mx_quantize(dtype, x, ldx, rows, K, image, nullptr, 1, stream);
}

int b2q_mx_dequantize(const uint8_t* image, int64_t rows, int64_t K, int dtype, void* y, int64_t ldy, b2q_stream_t stream) {
  const char* who = "b2q_mx_dequantize";
  int rc = check_mx_shape(who, rows, K);
  if (!rc) rc = check_mx_rows(who, "y", dtype, y, ldy, rows, K);
  if (rc || rows == 0) return rc;
  if (!image) return fail(B2Q_EINVAL, "%s: image is NULL", who);
  if (!aligned(y, 16) || (rows > 1 && ldy * mx_dtype_size(dtype) % 16) || !aligned(image, 128))
    return fail(B2Q_EALIGN, "%s: y and its row stride must be 16-byte aligned, the image 128-byte", who);
  const int stages = (int)mx_stages(K);
  unsigned grid;
  rc = grid_of(who, rows * stages * 16, &grid);
  if (rc) return rc;
  if (dtype == B2Q_DTYPE_F32)
    launch_maybe_pdl(mx_dequantize_kernel<float>, grid, 256, 0, stream, image, rows, (int)K, stages, static_cast<float*>(y), ldy);
  else if (dtype == B2Q_DTYPE_F16)
    launch_maybe_pdl(mx_dequantize_kernel<__half>, grid, 256, 0, stream, image, rows, (int)K, stages, static_cast<__half*>(y), ldy);
  else
    launch_maybe_pdl(mx_dequantize_kernel<__nv_bfloat16>, grid, 256, 0, stream, image, rows, (int)K, stages,
                     static_cast<__nv_bfloat16*>(y), ldy);
  return after_launch("mx_dequantize");
}

int b2q_mx_pack(const uint8_t* codes, const uint8_t* scales, int64_t experts, int64_t rows, int64_t K, uint8_t* image,
                b2q_stream_t stream) {
  const char* who = "b2q_mx_pack";
  int rc = check_mx_shape(who, rows, K);
  if (rc) return rc;
  if (experts < 1 || experts > kMaxExperts)
    return fail(B2Q_EINVAL, "%s: %lld experts (1..%lld)", who, (long long)experts, (long long)kMaxExperts);
  if (rows == 0) return B2Q_OK;
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
