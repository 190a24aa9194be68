// Internal interface of the tcgen05 tree attention (attn_tree_tc.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace eesd {

struct TreeGeom;
struct CacheGeom;

// The unit that a run's last piece begins and the next runs go on with (nrows = 0: none).
struct TcCut {
  int start, r0, nrows, h;    // its block's first token, first row of the row tile, rows, KV head
  int second, last;           // whether the piece is not the run's first; the last run with a piece of the unit
};

struct TcSchedule {
  int ctas;             // persistent CTAs
  int rows;             // query rows per tile: 128 or 256
  int tiles_max;        // row tiles of the largest block
  int entries;          // n_blocks * tiles_max
  int chunk_tiles;      // 0: equal runs; else key tiles per piece, cut at multiples of it
  TcCut* cuts;          // [ctas]
};

cudaError_t launch_attn_tree_tc(int fmt, int D, const TcSchedule& sc, const TreeGeom& g, const CacheGeom& c, const CUtensorMap& km,
                                const CUtensorMap& vm, const void* q, void* out, cudaStream_t s);

}  // namespace eesd
