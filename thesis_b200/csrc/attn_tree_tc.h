// Internal interface of the tcgen05 tree attention (attn_tree_tc.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace eesd {

struct TreeGeom;
struct CacheGeom;

// The unit that a run's last piece begins and the next runs go on with (e < 0: none).
struct TcCut {
  long long u0;               // flat position of the unit (behind the last run: the length of the flat axis)
  int e, h, second, tiles;    // entry, KV head, whether the piece is not the run's first, key tiles
};

struct TcSchedule {
  int ctas;             // persistent CTAs
  int rows;             // query rows per tile: 128 or 256
  int tiles_max;        // row tiles of the largest block
  int entries;          // n_blocks * tiles_max
  int chunk_tiles;      // 0: equal runs; else key tiles per piece, cut at multiples of it
  TcCut* cuts;          // [ctas + 1]
};

cudaError_t launch_attn_tree_tc(int fmt, int D, const TcSchedule& sc, const TreeGeom& g, const CacheGeom& c, const CUtensorMap& km,
                                const CUtensorMap& vm, const void* q, void* out, cudaStream_t s);

}  // namespace eesd
