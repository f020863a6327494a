// Sizes of the MXFP4 kernels that the host decides on: the operand image, and how the one-launch product is cut (host code
// alone, so that it can be compiled and looked over without CUDA).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace b2q {

// An operand image: tiles of 128 rows by stages of 256 values. A stage of a tile is one run of 17408 bytes: 128 rows of 128
// bytes of codes, then the scales of its 8 blocks a row (see mx_device.cuh).
constexpr int kMxRows = 128, kMxStage = 256;
constexpr int kMxCodes = kMxRows * kMxStage / 2, kMxScales = kMxRows * kMxStage / 32, kMxBytes = kMxCodes + kMxScales;

// The product of up to 4 rows in one launch (mx_gemv.cu).
constexpr int kGemvRing = 8;                            // stages of weights in shared memory at the most
constexpr int kGemvRows = 4, kGemvXStage = 8 * 128;     // rows of x; bytes of a stage of them, a whole group of 8
constexpr uint32_t kGemvScaleW = 32, kGemvScaleX = 48;  // columns: accumulators 2 x 16, weight scales 2 x 8, then 4 a stage of x
constexpr size_t kGemvSmem = 214 * 1024;

// A ring's stages are numbered as they are asked for: stage i lies in slot i % ring, and its arrival is phase i / ring of the slot's
// barrier. Of `issued` stages the ones from here on, a slot's last each, may be under way still.
constexpr uint32_t first_under_way(uint32_t issued, uint32_t ring) { return issued > ring ? issued - ring : 0; }

struct GemvPlan {
  int ranks, nk, ring;  // CTAs in a cluster, the most stages one has, stages of its ring
  int columns;          // of tensor memory
  size_t smem;
};

// Whether and how the kernel takes `rows` rows of x with `used` experts of `row_tiles` tiles, on a GPU of `sms` SMs.
inline bool plan_gemv(int64_t rows, int64_t used, int64_t row_tiles, int64_t stages, int sms, GemvPlan* p) {
  if (rows < 1 || rows > kGemvRows || used * row_tiles > INT32_MAX / 2) return false;
  int ranks = 1;
  while (ranks < 8 && used * row_tiles * ranks * 2 <= sms && stages >= ranks * 2) ranks *= 2;
  const int64_t nk = (stages + ranks - 1) / ranks;
  if (nk > (512 - (int)kGemvScaleX) / 4 - 1) return false;
  const size_t x = (size_t)(nk + 1) * kGemvXStage + nk * 512 + 1024;  // 1024: the ring is aligned to that
  // a ring that leaves room for the next kernel's CTA beside this one, or else for all that an SM has
  const size_t half = 104 * 1024, all = kGemvSmem;
  size_t ring = x + 4 * kMxBytes <= half ? (half - x) / kMxBytes : x + 3 * kMxBytes <= all ? (all - x) / kMxBytes : 0;
  if (ring == 0) return false;
  ring = std::min<size_t>(std::min<size_t>(ring, kGemvRing), std::max<int64_t>(nk, 2));
  // As many columns as the scales take (and four that stay free after the last) and no more: whatever calls an SM's shared
  // memory has room for at once, its tensor memory has too.
  int columns = 64;
  while (columns < (int)kGemvScaleX + 4 * nk + 4) columns *= 2;
  *p = {ranks, (int)nk, (int)ring, columns, x + ring * kMxBytes};
  return true;
}

}  // namespace b2q
