// Host-side internals shared by the KV cache and attention translation units: argument checks, the parameter block of
// the attention kernels and the launchers that the dispatcher picks from.
#pragma once

#include <atomic>

#include "b2q_internal.h"

namespace b2q {

constexpr int kErrSlot = 2;  // device error word: a slot beyond the cache
constexpr int kErrPage = 3;  // device error word: a token whose page is outside the table or the cache
constexpr int kErrQueries = 4;  // device error word: query tokens past the tiles that max_q gave a sequence

inline int dtype_size(int dtype) { return dtype == B2Q_DTYPE_F32 ? 4 : 2; }

// The checks of a cache descriptor that every entry point makes (kv_cache.cu).
int check_kv_cache(const char* who, const b2q_kv_cache* c);

// Lets `kernel` (told apart by the caller's own `done` word) take `bytes` of shared memory, once a device.
int allow_smem_once(const void* kernel, int bytes, std::atomic<unsigned long long>& done);

// A tile that several CTAs worked on, told by the CTA that ended it: the CTA that began it (-1: no such tile), the tile's
// rows, its first row and head, and its sequence's first query token.
struct AttnJoin {
  int first, rows, row0, head0, q0;
};

struct AttnParams {
  const void* q;
  void* out;
  float* lse;
  const uint8_t *kq, *vq;
  const uint16_t *ks, *vs;
  const int32_t *table, *lens, *cu_q, *prefix, *starts;
  const float* slopes;
  float* part_o;    // [2 a CTA][rows of a tile][dim] outputs, not divided, of tiles that cross CTAs' shares
  float2* part_m;   // [2 a CTA][rows of a tile] their reference exponent and sum
  AttnJoin* joins;  // [CTAs]
  int64_t q_st, q_sh, T, table_stride, pages;
  int table_pages, batch, q_heads, heads, group, page_shift, row_tiles, window, dtype;
  int tile_cost;  // tensor-core kernels: what beginning a tile costs, in blocks of keys
  float scale, softcap;
};

// A device error word lives in each translation unit whose kernels set one; b2q_device_error reads them all.
int kv_cache_error(int* code, int clear);
int kv_attention_q4_error(int* code, int clear);
int kv_attention_q8_error(int* code, int clear);
int kv_attention_tc_q4_error(int* code, int clear);
int kv_attention_tc_q8_error(int* code, int clear);

// Streaming kernels by format: `rows` is 8 or 16 query rows a tile, max_len bounds the lengths from above.
int launch_attention_q4(const AttnParams& p, int dim, int rows, int sms, int64_t max_len, cudaStream_t stream);
int launch_attention_q8(const AttnParams& p, int dim, int rows, int sms, int64_t max_len, cudaStream_t stream);
// Tensor-core kernels by format, for tiles of kTcRows (heads of 256: half as many) query rows; 16-bit queries only.
int launch_attention_tc_q4(const AttnParams& p, int dim, int sms, cudaStream_t stream);
int launch_attention_tc_q8(const AttnParams& p, int dim, int sms, cudaStream_t stream);
constexpr int kTcRows = 256;
constexpr int kMaxCtasPerSm = 3;  // the workspace holds parts for so many

}  // namespace b2q
