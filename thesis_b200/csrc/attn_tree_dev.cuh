// Device code that the tree attention kernels share: geometry, visibility, packing.
#pragma once

#include "cache.cuh"

namespace eesd {

struct TreeGeom {
  int n_heads, G;
  int n_tokens, max_nodes, max_ctx, words;
  const int32_t* blk;
  const uint64_t* mask;
  int ld_q;
  float scale;
  int* status;
  uint32_t spin;       // poll limit of the pipeline waits
  int chunk, splits;   // keys per CTA; key ranges of the longest row
  bool sort;           // long blocks first
  float* part_o;       // [n_tokens, Hq, splits, D] normalised partial outputs
  float2* part_ml;     // [n_tokens, Hq, splits] (max in the log2 domain, sum)
};

struct BlockInfo {
  int start, T, row, ctx;
};
// Reads block b; false where it does not fit the tokens, the maxima or the cache.
__device__ __forceinline__ bool block_fits(const TreeGeom& g, const CacheGeom& c, int b, BlockInfo& i) {
  const int4 v = *reinterpret_cast<const int4*>(g.blk + 4 * b);
  i.start = v.x, i.T = v.y, i.row = v.z, i.ctx = v.w;
  return i.start >= 0 && i.T > 0 && i.T <= g.max_nodes && i.start <= g.n_tokens - i.T && i.row >= 0 && i.row < c.max_batch &&
         i.ctx >= 0 && i.ctx <= min(g.max_ctx, c.max_seq) - i.T;
}
// The same, and a status bit from one thread.
__device__ __forceinline__ bool load_block(const TreeGeom& g, const CacheGeom& c, int b, BlockInfo& i) {
  const bool ok = block_fits(g, c, b, i);
  if (!ok && threadIdx.x == 0) set_status(g.status, kStatusBadIndex);
  return ok;
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
template <int FMT> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (FMT == EESD_KV_MODEL) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
// bf16 pair with its non-finite elements replaced by zero
__device__ __forceinline__ uint32_t drop_nonfinite(uint32_t v, bool& hit) {
  const bool lo = (v & 0x7f80u) == 0x7f80u, hi = (v & 0x7f800000u) == 0x7f800000u;
  hit = hit || lo || hi;
  return (lo ? 0u : v & 0xffffu) | (hi ? 0u : v & 0xffff0000u);
}

// Which of the 32 nodes j0 .. j0 + 31 a node sees (bit i: node j0 + i); negative nodes are committed slots.
// mask: the node's words, or null for causal blocks.
__device__ __forceinline__ uint32_t sees32(const uint64_t* mask, int words, int node, int j0) {
  if (!mask) {
    const int n = node - j0 + 1;
    return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1;
  }
  if (j0 <= -32) return ~0u;
  if (j0 < 0) return (uint32_t)(mask[0] << -j0) | ((1u << -j0) - 1);
  const int w = j0 >> 6, sh = j0 & 63;
  uint64_t v = w < words ? mask[w] >> sh : 0;
  if (sh > 32 && w + 1 < words) v |= mask[w + 1] << (64 - sh);
  return (uint32_t)v;
}

}  // namespace eesd
