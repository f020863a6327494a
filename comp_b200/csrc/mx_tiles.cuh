// How the persistent MXFP4 products cut their work into tiles: `units` of weight rows by TN rows of x of one expert.
#pragma once

#include "mx_tc.cuh"

namespace b2q {

// A tile: its weight rows, its rows of y, and where its rows of x lie in the image.
struct TileAt {
  int e, rt;    // expert, and which of the units of weight rows
  int x_tile;   // 128-row tile of the image of x that holds its first row
  int row0;     // first row of y
  int sub, n;   // first row within x_tile, rows
  bool again;   // other tiles read the same weights
};

// Where the experts' rows and tiles begin, in shared memory: [experts + 1] rows of y, tiles of TN rows, tiles of the image.
struct Experts {
  const int *rows, *tiles, *image;
};

template <int TN>
__device__ __forceinline__ TileAt tile_at(const MxGemm& g, const Experts& x, int t, int units) {
  TileAt r;
  int e = 0, local = t, rows = (int)g.rows, count = (rows + TN - 1) / TN, base = 0, tile0 = 0;
  if (g.offsets) {
    int lo = 0, hi = g.experts;  // the expert whose tiles hold t: tiles[e] * units <= t < tiles[e + 1] * units
    const int nth = t / units;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (x.tiles[mid] <= nth) lo = mid;
      else hi = mid;
    }
    e = lo;
    local = t - x.tiles[e] * units;
    count = x.tiles[e + 1] - x.tiles[e];
    base = x.rows[e], rows = x.rows[e + 1] - base, tile0 = x.image[e];
  }
  // the tiles of the same weights follow one another, so that those are read from memory once
  const int rt = local / count, at = (local - rt * count) * TN;
  r.e = e, r.rt = rt, r.x_tile = tile0 + (at >> 7), r.sub = at & 127;
  r.row0 = base + at, r.n = min(TN, rows - at), r.again = count > 1;
  return r;
}

// The table of an MxGemm in shared memory (3 (experts + 1) words), made by all THREADS threads of a CTA, and the number of
// tiles; a barrier later all may read them. scratch: a word a warp.
template <int TN, int THREADS>
__device__ __forceinline__ Experts count_tiles(const MxGemm& g, int* table, int* scratch, int* tiles, int units) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (g.offsets) {  // THREADS experts at a time
    int before = 0;
    for (int e0 = 0; e0 <= g.experts; e0 += THREADS) {
      const int e = e0 + threadIdx.x;
      const int row = e <= g.experts ? g.offsets[e] : 0, rows = e < g.experts ? g.offsets[e + 1] - row : 0;
      const int mine = (rows + TN - 1) / TN;
      if (e <= g.experts) table[e] = row, table[2 * (g.experts + 1) + e] = g.tiles[e];
      int sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      if (lane == 31) scratch[warp] = sum;
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int i = 0; i < THREADS / 32; ++i) {
        if (i < warp) sum += scratch[i];
        all += scratch[i];
      }
      if (e < g.experts) table[g.experts + 1 + e] = before + sum - mine;
      before += all;
      __syncthreads();
    }
    if (threadIdx.x == 0) table[2 * g.experts + 1] = before, *tiles = before * units;
  } else if (threadIdx.x == 0) {
    *tiles = (int)((g.rows + TN - 1) / TN) * units;
  }
  return {table, table + g.experts + 1, table + 2 * (g.experts + 1)};
}

}  // namespace b2q
