// Host-side internals shared by the MXFP4 and expert translation units: argument checks, launchers.
#pragma once

#include "b2q_internal.h"
#include "mx_plan.h"

namespace b2q {

constexpr int kErrExpert = 5;  // device error word: an expert's number beyond the experts

constexpr int64_t kMaxExperts = 1024, kMaxTop = 32;

inline int64_t mx_tiles(int64_t rows) { return (rows + kMxRows - 1) / kMxRows; }
inline int64_t mx_stages(int64_t K) { return (K + kMxStage - 1) / kMxStage; }

inline int mx_dtype_size(int dtype) { return dtype == B2Q_DTYPE_F32 ? 4 : 2; }

// Rows and values of an image that every entry point checks (mx_quant.cu).
int check_mx_shape(const char* who, int64_t rows, int64_t K);
int check_mx_rows(const char* who, const char* name, int dtype, const void* x, int64_t ldx, int64_t rows, int64_t K);

// Quantizes x into an image: row r goes to the image rows dest[r * fan + j], j < fan (negative: nowhere), or without dest to its
// place among operands of `each` rows.
int launch_mx_quantize(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t each, int64_t K, uint8_t* image,
                       const int32_t* dest, int fan, cudaStream_t stream);

struct MxGemm {
  const uint8_t *w, *x;    // images: the weights of all experts, one after the other; the rows
  void* y;
  const int32_t* offsets;  // [experts + 1] where each expert's rows begin in y (null: one expert with `rows` rows)
  const int32_t* tiles;    // [experts + 1] and in the image x, in tiles of 128 rows
  int64_t ldy, rows;       // rows of y: without offsets all there are, with them at most so many
  int N, row_tiles, stages, experts, dtype;
  int early;               // the weights, offsets and tiles may be read before the preceding kernel has ended
};
int launch_mx_gemm(const MxGemm& g, cudaStream_t stream);

// Up to 4 rows of x, quantized by the kernel itself.
struct MxGemv {
  const uint8_t* w;
  const void* x;
  void* y;
  const int32_t *offsets, *order;  // of a plan (null: one expert)
  int64_t ldx, ldy, rows, choices, experts, N, K;
  int x_dtype, dtype, top;         // top: choices a token where x has a row a token (0: x has the sorted rows)
};
bool mx_gemv_takes(int64_t rows, int64_t choices, int64_t experts, int64_t N, int64_t K);
int launch_mx_gemv(const MxGemv& a, cudaStream_t stream);

// A translation unit's device error word (b2q_device_error reads them all).
int mx_gemm_error(int* code, int clear);
int mx_gemv_error(int* code, int clear);
int experts_error(int* code, int clear);

}  // namespace b2q
