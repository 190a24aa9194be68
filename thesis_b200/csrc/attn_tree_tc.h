// Internal interface of the tcgen05 tree attention (attn_tree_tc.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace eesd {

struct TreeGeom;
struct CacheGeom;

struct TcSchedule {
  int ctas;             // persistent CTAs
  int rows;             // query rows per tile: 128 or 256
  int tiles_max;        // row tiles of the largest block
  int entries;          // n_blocks * tiles_max
  int chunk_tiles;      // 0: equal runs; else key tiles per piece, cut at multiples of it
  long long* table;     // [entries + 1] flat position of every entry, and the total
};

cudaError_t launch_attn_tree_tc(int fmt, int D, const TcSchedule& sc, const TreeGeom& g, const CacheGeom& c, const CUtensorMap& km,
                                const CUtensorMap& vm, int n_blocks, const void* q, void* out, cudaStream_t s);

}  // namespace eesd
