// Attention of tree nodes and causal chains over a KV cache in the model dtype or in 8 bits, and its C entry.
//
// o[r] = sum_j p_rj v_j / sum_j p_rj,  p_rj = exp(s_rj - max_j s_rj),  s_rj = q_r . k_j / sqrt(D), over the
// slots j that row r sees.  Rows are (node, query head of the KV group) pairs, r = node * G + head, so one
// read of a key serves all heads of its group and all nodes of the block.
#include <math.h>

#include "attn_tree.h"
#include "cache.cuh"

namespace eesd {
namespace {

struct TreeGeom {
  int n_heads, G;
  int n_tokens, max_nodes, max_ctx, words;
  const int32_t* blk;
  const uint64_t* mask;
  int ld_q;
  float scale;
  int* status;
};

struct BlockInfo {
  int start, T, row, ctx;
};
// Reads block b; false (and a status bit, from one thread) where it does not fit the tokens, the maxima or the cache.
__device__ __forceinline__ bool load_block(const TreeGeom& g, const CacheGeom& c, int b, BlockInfo& i) {
  const int4 v = *reinterpret_cast<const int4*>(g.blk + 4 * b);
  i.start = v.x, i.T = v.y, i.row = v.z, i.ctx = v.w;
  const bool ok = i.start >= 0 && i.T > 0 && i.T <= g.max_nodes && i.start <= g.n_tokens - i.T && i.row >= 0 &&
                  i.row < c.max_batch && i.ctx >= 0 && i.ctx <= min(g.max_ctx, c.max_seq) - i.T;
  if (!ok && threadIdx.x == 0) set_status(g.status, kStatusBadIndex);
  return ok;
}
__device__ __forceinline__ bool node_sees(const TreeGeom& g, const BlockInfo& i, int node, int j) {
  if (!g.mask) return j <= node;
  return j < 64 * g.words && (g.mask[(size_t)(i.start + node) * g.words + (j >> 6)] >> (j & 63) & 1);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

template <typename T, int FMT> __device__ __forceinline__ float cache_value(const void* p, const uint8_t* e, size_t slot, int D, int d) {
  if constexpr (FMT == EESD_KV_MODEL) {
    return to_f(static_cast<const T*>(p)[slot * D + d]);
  } else {
    uint32_t lo, hi;
    unpack4<FMT>(static_cast<const uint8_t*>(p)[slot * D + d], lo, hi);
    return half2_to_float2(lo).x * kHalfUnit<FMT> * exp_scale(e[slot]);
  }
}

// fp32 path: scalar online softmax, one warp per row (8 rows each), 32-key tiles in shared memory.
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(128) attn_tree_simt_kernel(TreeGeom g, CacheGeom c, const T* __restrict__ q, T* __restrict__ out) {
  pdl_trigger();
  pdl_wait();
  constexpr int KT = 32, DP = D + 1, ND = D / 32, MAXR = 8;
  extern __shared__ float sm[];
  float* Qs = sm;                   // [32][D]
  float* Ks = Qs + 32 * D;          // [KT][DP]
  float* Vs = Ks + KT * DP;         // [KT][D]
  BlockInfo bi;
  if (!load_block(g, c, blockIdx.z, bi)) return;
  const int kvh = blockIdx.y, r0 = blockIdx.x * 32;
  const int nrows = min(32, bi.T * g.G - r0);
  if (nrows <= 0) return;
  const int last = (r0 + nrows - 1) / g.G;                                 // last node of the tile
  const int n_keys = bi.ctx + (g.mask ? bi.T : last + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int idx = threadIdx.x; idx < nrows * D; idx += blockDim.x) {
    const int r = r0 + idx / D, d = idx % D;
    Qs[idx] = to_f(q[(size_t)(bi.start + r / g.G) * g.ld_q + (kvh * g.G + r % g.G) * D + d]);
  }
  const size_t slot0 = cache_slot(c, bi.row, kvh, 0);
  float m[MAXR], l[MAXR], acc[MAXR][ND];
#pragma unroll
  for (int i = 0; i < MAXR; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < ND; ++e) acc[i][e] = 0.f;
  }
  for (int k0 = 0; k0 < n_keys; k0 += KT) {
    __syncthreads();
    for (int idx = threadIdx.x; idx < KT * D; idx += blockDim.x) {
      const int j = idx / D, d = idx % D;
      const bool in = k0 + j < n_keys;
      Ks[j * DP + d] = in ? cache_value<T, FMT>(c.k, c.ke, slot0 + k0 + j, D, d) : 0.f;
      Vs[j * D + d] = in ? cache_value<T, FMT>(c.v, c.ve, slot0 + k0 + j, D, d) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MAXR; ++i) {
      const int r = warp + 4 * i;
      if (r < nrows) {
        const int node = (r0 + r) / g.G, key = k0 + lane;
        const bool sees = key < n_keys && (key < bi.ctx || node_sees(g, bi, node, key - bi.ctx));
        float s = -INFINITY;
        if (sees) {
          float dot = 0.f;
          for (int d = 0; d < D; ++d) dot = fmaf(Qs[r * D + d], Ks[lane * DP + d], dot);
          s = dot * g.scale;
        }
        const float mn = fmaxf(m[i], warp_max(s));
        const float ms = mn == -INFINITY ? 0.f : mn;
        const float corr = expf(m[i] - ms);
        const float p = sees ? expf(s - ms) : 0.f;
        l[i] = l[i] * corr + warp_sum(p);
        const unsigned any = __ballot_sync(0xffffffffu, sees);
#pragma unroll
        for (int e = 0; e < ND; ++e) acc[i][e] *= corr;
#pragma unroll 4
        for (int j = 0; j < KT; ++j) {
          const float pj = __shfl_sync(0xffffffffu, p, j);
          if (any >> j & 1) {          // an unseen slot's V is not touched: it may be NaN
#pragma unroll
            for (int e = 0; e < ND; ++e) acc[i][e] = fmaf(pj, Vs[j * D + e * 32 + lane], acc[i][e]);
          }
        }
        m[i] = mn;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MAXR; ++i) {
    const int r = warp + 4 * i;
    if (r < nrows) {
      const int R = r0 + r;
      const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];                   // a node that sees nothing: zeros
      T* o = out + ((size_t)(bi.start + R / g.G) * g.n_heads + kvh * g.G + R % g.G) * D;
#pragma unroll
      for (int e = 0; e < ND; ++e) o[e * 32 + lane] = from_f<T>(acc[i][e] * inv);
    }
  }
}

template <typename T, int FMT, int D>
cudaError_t launch_simt(const TreeGeom& g, const CacheGeom& c, int n_blocks, const void* q, void* out, cudaStream_t s) {
  const dim3 grid((g.max_nodes * g.G + 31) / 32, c.n_kv_heads, n_blocks);
  constexpr size_t smem = (32 * D + 32 * (D + 1) + 32 * D) * 4;
  const cudaError_t e = cudaFuncSetAttribute(attn_tree_simt_kernel<T, FMT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(attn_tree_simt_kernel<T, FMT, D>, grid, dim3(128), smem, s, g, c, static_cast<const T*>(q), static_cast<T*>(out));
}
template <typename T>
cudaError_t launch_simt_fmt(int fmt, int D, const TreeGeom& g, const CacheGeom& c, int nb, const void* q, void* out, cudaStream_t s) {
  switch (fmt * 2 + (D == 128)) {
    case 0: return launch_simt<T, EESD_KV_MODEL, 64>(g, c, nb, q, out, s);
    case 1: return launch_simt<T, EESD_KV_MODEL, 128>(g, c, nb, q, out, s);
    case 2: return launch_simt<T, EESD_KV_E4M3, 64>(g, c, nb, q, out, s);
    case 3: return launch_simt<T, EESD_KV_E4M3, 128>(g, c, nb, q, out, s);
    case 4: return launch_simt<T, EESD_KV_INT8, 64>(g, c, nb, q, out, s);
    default: return launch_simt<T, EESD_KV_INT8, 128>(g, c, nb, q, out, s);
  }
}

int check_attn(int dtype, const EesdKvCache* c, int layer, const EesdTree* t, int n_heads, int split_keys) {
  int rc = check_cache("attn_tree", dtype, c, layer);
  if (!rc) rc = check_tree("attn_tree", t);
  if (rc) return rc;
  if (n_heads <= 0 || n_heads % c->n_kv_heads) return fail_arg(EESD_ERR_ARG, "attn_tree: heads %d / %d", n_heads, c->n_kv_heads);
  if (split_keys < 0 || split_keys % 256) return fail_arg(EESD_ERR_ARG, "attn_tree: split_keys %d (0 or a multiple of 256)", split_keys);
  if (t->n_tokens && t->n_blocks && t->max_ctx > c->max_seq)
    return fail_arg(EESD_ERR_ARG, "attn_tree: max_ctx %d > max_seq %d", t->max_ctx, c->max_seq);
  return EESD_OK;
}

}  // namespace
}  // namespace eesd

using namespace eesd;

extern "C" {

size_t eesd_attn_tree_workspace_bytes(int dtype, const EesdKvCache* c, const EesdTree* t, int n_heads, int split_keys) {
  if (check_attn(dtype, c, 0, t, n_heads, split_keys)) return 0;
  return 256;
}

int eesd_attn_tree(int dtype, const EesdKvCache* c, int layer, const EesdTree* t, const void* q, int ld_q, int n_heads, void* out,
                   int split_keys, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  int rc = check_attn(dtype, c, layer, t, n_heads, split_keys);
  if (rc) return rc;
  if (t->n_tokens == 0 || t->n_blocks == 0) return EESD_OK;
  if (!q || !out) return fail_arg(EESD_ERR_ARG, "attn_tree: null argument");
  if (ld_q % 8 || ld_q < n_heads * c->head_dim)
    return fail_arg(EESD_ERR_ARG, "attn_tree: ld_q %d (a multiple of 8, at least Hq D)", ld_q);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(t->blk)) & 15)
    return fail_arg(EESD_ERR_ARG, "attn_tree: q, out and blk must be 16-byte aligned");
  const size_t need = eesd_attn_tree_workspace_bytes(dtype, c, t, n_heads, split_keys);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255))
    return fail_arg(EESD_ERR_ARG, "attn_tree: workspace %zu < %zu bytes, or not 256-byte aligned", workspace_bytes, need);
  if ((rc = check_stream("attn_tree", stream))) return rc;
  const CacheGeom cg = cache_layer(c, dtype, layer);
  const TreeGeom g{n_heads, n_heads / c->n_kv_heads, t->n_tokens, t->max_nodes, t->max_ctx, t->words, t->blk, t->mask, ld_q,
                   1.f / sqrtf((float)c->head_dim), status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == EESD_BF16 ? launch_simt_fmt<bf16>(c->format, c->head_dim, g, cg, t->n_blocks, q, out, s)
                                           : launch_simt_fmt<float>(c->format, c->head_dim, g, cg, t->n_blocks, q, out, s);
  return e == cudaSuccess ? EESD_OK : fail_arg(EESD_ERR_CUDA, "attn_tree: launch: %s", cudaGetErrorString(e));
}

}  // extern "C"
