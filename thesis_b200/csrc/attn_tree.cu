// Attention of tree nodes and causal chains over a KV cache in the model dtype or in 8 bits, and its C entry.
//
// o[r] = sum_j p_rj v_j / sum_j p_rj,  p_rj = exp(s_rj - max_j s_rj),  s_rj = q_r . k_j / sqrt(D), over the
// slots j that row r sees.  Rows are (node, query head of the KV group) pairs, r = node * G + head, so one
// read of a key serves all heads of its group and all nodes of the block.
#include <math.h>

#include <algorithm>

#include "attn_tree.h"
#include "attn_tree_dev.cuh"
#include "attn_tree_tc.h"
#include "gemm_tc.h"

namespace eesd {
namespace {

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

// ---------------------------------------------------------------- small row tiles: mma.sync
// One CTA per (row tile of 8 NT rows, KV head, key range of a block): a few query rows against a stream of keys,
// bound by the bytes of K and V.  Its 4 warps are independent: warp w takes every fourth group of KG keys (16 .. 64,
// 8 KB of K and V) through a TMA ring of its own, so nothing in the key loop waits for another warp; the warps'
// running (max, sum, output) meet once at the end.
//
// The products are the transposed ones, S^T = K Q^T and O^T = V^T P^T on m16n8k16: 16 keys (or dims) fill the M side,
// and the query rows, 4 to 32 of them, are the N side in steps of 8, so few rows cost few products and few registers
// (O^T is 32 registers per 8 rows of 128 dims).  A thread has S of two rows; a row's maximum would be a reduction over 8
// lanes, so it is only taken when some score is 2^8 above the running reference.  P^T becomes an operand by
// transposing its 8 x 8 blocks between lanes (movmatrix).
//
// Both products may order their contraction index, and O^T its rows, as they like, which the 8-bit formats use:
// thread (g, t) = (lane / 4, lane % 4) takes the dims [t D/4, (t + 1) D/4) of keys g and g + 8 as K fragments and the
// dims [g D/8, (g + 1) D/8) of keys 2t, 2t + 1, 2t + 8, 2t + 9 as V fragments, so K and V come from shared memory as
// 16-byte words and turn into f16 pairs in registers, without a transpose.  The values' powers of two never touch the
// operands: K's scale multiplies the score, V's the weight (relative to the row's largest weight x scale so far, er, as
// the score is to the running maximum), a power of two of each q row its f16 form.  Weights are rounded to f16 (2^-11; a bf16 cache:
// to bf16, 2^-8, the type of V), sums and outputs are fp32.
//
// Measured (32 query and 8 KV heads of 128): 64 trees of 5 nodes at 129 to 1023 slots over bf16 36 us, 4.4 TB/s, 68 % of the
// copy rate; 64 single tokens over int8 25 us, 3.1 TB/s (the conversion of the bytes and a unit's start and end take the
// issue slots); 8 trees of 17 nodes at 501 to 2013 slots, 32 KV heads over bf16, 50 us, 3.4 TB/s.
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <int FMT> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (FMT == EESD_KV_MODEL)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D, int FMT, int NT> struct MmaShape {
  static constexpr int kEb = FMT == EESD_KV_MODEL ? 2 : 1;
  static constexpr int KG = 4096 / (D * kEb);          // keys per group: 4 KB of K, 4 KB of V
  // (three CTAs with two stages a warp or two with three: where the registers of three would spill)
  static constexpr int CTAS = NT == 4 || (NT == 3 && D == 128 && kEb == 1) ? 2 : 3;   // resident CTAs per SM, by registers
  static constexpr int NS = CTAS == 2 ? 3 : 2;         // ring stages per warp
  static constexpr int ROWS = 8 * NT;
  static constexpr int STAGE = 8192;
  static constexpr int Q_BYTES = ROWS * D * 2;         // fragment order: [n-tile][k-step][lane] pairs of words
  static constexpr int OLD = D + 4;
  static constexpr size_t smem = 1024 + 4 * NS * STAGE + Q_BYTES + 4 * NS * 128 + ROWS * 32 + ROWS * 4 + 4 * NS * 8 + 16;
  static_assert((4 * ROWS * OLD + 12 * ROWS) * 4 <= 4 * NS * STAGE, "the merge does not fit the stage memory");
};

// The block that grid layer z works on: the z-th longest.  CTAs start in grid order, so the long contexts run first and the
// short ones fill the SMs that are done: 64 single tokens at 129 to 1023 slots over int8 25 us instead of 28, 5-node trees
// over bf16 36 instead of 41.  It costs up to 2 us, so only grids that leave SMs two CTAs and more do it; beyond kSorted
// blocks the order given evens out by itself.
constexpr int kSorted = 128;                                             // a CTA's threads
__device__ __forceinline__ int longest_first(const TreeGeom& g) {
  __shared__ alignas(16) unsigned long long key[kSorted];
  __shared__ int pick;
  const int n = gridDim.z, t = threadIdx.x;                             // one thread per block of the batch
  if (!g.sort) return blockIdx.z;
  unsigned long long mine = 0;                                          // T + ctx, and the earlier block first among equals
  if (t < n) {
    const int4 v = *reinterpret_cast<const int4*>(g.blk + 4 * t);
    mine = (unsigned long long)((unsigned)v.y + (unsigned)v.w) << 8 | (unsigned)(255 - t);
  }
  key[t] = mine;
  __syncthreads();
  if (t < n) {
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; j += 2) {
      const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(key + j);
      rank += (v.x > mine) + (v.y > mine);
    }
    if (rank == (int)blockIdx.z) pick = t;
  }
  __syncthreads();
  return pick;
}

constexpr float kNone = -3.402823466e38f;                                // the maximum of no scores: finite, so that -inf minus it is no NaN

template <int D, int FMT, int NT>
__global__ void __launch_bounds__(128, MmaShape<D, FMT, NT>::CTAS)
    attn_tree_mma_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, TreeGeom g, CacheGeom c,
                         const bf16* __restrict__ q, bf16* __restrict__ out) {
  using P = MmaShape<D, FMT, NT>;
  constexpr bool Q8 = FMT != EESD_KV_MODEL;
  constexpr int KG = P::KG, NS = P::NS, ROWS = P::ROWS, OLD = P::OLD, MD = D / 16;   // 16-dim steps of both products
  constexpr int HALF = 4096;                           // K bytes (then V bytes) of a stage
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  pdl_trigger();
  pdl_wait();
  extern __shared__ uint8_t smem8[];
  uint8_t* sm = smem8 + (-smem_u32(smem8) & 1023);                      // an offset: the compiler still knows it as shared memory
  uint8_t* stages = sm;                                                 // [4 warps][NS][K | V]
  uint8_t* qs = sm + 4 * NS * P::STAGE;
  uint8_t* exps = qs + P::Q_BYTES;                                      // [4][NS][K bytes 64 | V bytes 64]
  uint64_t* masks = reinterpret_cast<uint64_t*>(exps + 4 * NS * 128);   // [ROWS][4], a row's node
  float* qscale = reinterpret_cast<float*>(masks + ROWS * 4);           // [ROWS] power of two taken out of the q row
  uint64_t* full = reinterpret_cast<uint64_t*>(qscale + ROWS);          // [4][NS]
  volatile int* flags = reinterpret_cast<volatile int*>(full + 4 * NS);   // [0] a wait gave up, [1] a non-finite V was dropped

  BlockInfo bi;
  if (!load_block(g, c, longest_first(g), bi)) return;
  const int kvh = blockIdx.y % c.n_kv_heads, r0 = blockIdx.y / c.n_kv_heads * ROWS;
  const int nrows = min(ROWS, bi.T * g.G - r0);
  if (nrows <= 0) return;
  const int first = r0 / g.G, last = (r0 + nrows - 1) / g.G;            // the tile's nodes
  const int n_keys = bi.ctx + (g.mask ? bi.T : last + 1);
  const int k_lo = blockIdx.x * g.chunk, k_hi = min(n_keys, k_lo + g.chunk);
  if (k_lo >= n_keys) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  const int all_see = bi.ctx + (g.mask ? 0 : first + 1);                // slots below this are seen by every row
  const int n_groups = (k_hi - k_lo + KG - 1) / KG;
  const int my_groups = warp < n_groups ? (n_groups - warp + 3) / 4 : 0;
  const int slot0 = (int)cache_slot(c, bi.row, kvh, 0);                 // fits: the entry point bounds the layer's slots

  const uint32_t st0 = smem_u32(stages) + warp * NS * P::STAGE;
  const uint32_t fb0 = smem_u32(full + warp * NS);
  uint8_t* const ex0 = exps + warp * NS * 128;
  auto issue = [&](int i) {                                             // lane 0: this warp's i-th group
    const int s = i % NS, key = k_lo + (warp + 4 * i) * KG;
    const uint32_t fb = fb0 + s * 8, dst = st0 + s * P::STAGE;
    if constexpr (Q8) {
      const uint32_t eb = min(KG, c.max_seq - key), ex = smem_u32(ex0 + s * 128);   // max_seq % 16 == 0 and key % 16 == 0
      mbar_arrive_expect_tx(fb, P::STAGE + 2 * eb);
      tma_load_2d(dst, &kmap, 0, slot0 + key, fb);
      tma_load_2d(dst + HALF, &vmap, 0, slot0 + key, fb);
      bulk_g2s(ex, c.ke + slot0 + key, eb, fb);
      bulk_g2s(ex + 64, c.ve + slot0 + key, eb, fb);
    } else {
      mbar_arrive_expect_tx(fb, P::STAGE);
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        tma_load_2d(dst + h * KG * 128, &kmap, h * 64, slot0 + key, fb);
        tma_load_2d(dst + HALF + h * KG * 128, &vmap, h * 64, slot0 + key, fb);
      }
    }
  };
  if (lane == 0) {
    for (int s = 0; s < NS; ++s) mbar_init(fb0 + s * 8, 1);
    fence_mbar_init();
    for (int i = 0; i < NS && i < my_groups; ++i) issue(i);
  }
  if (threadIdx.x == 0) flags[0] = flags[1] = 0;
  // q rows of the tile (zeros behind nrows) and their nodes' masks, all loads at once: 4 threads per row
  {
    constexpr int V = D / 32;                                           // 16-byte chunks per thread, 4 apart
    const int r = threadIdx.x / 4, part = threadIdx.x % 4, R = r0 + r;
    const bool in = r < nrows;
    const int node = in ? R / g.G : 0;
    const bf16* src = q + (size_t)(bi.start + node) * g.ld_q + (kvh * g.G + (in ? R - node * g.G : 0)) * D;
    uint4 u[V];
#pragma unroll
    for (int i = 0; i < V; ++i) u[i] = in ? *reinterpret_cast<const uint4*>(src + (part + i * 4) * 8) : make_uint4(0, 0, 0, 0);
    const uint64_t mk = g.mask && in && part < g.words ? g.mask[(size_t)(bi.start + node) * g.words + part] : 0ull;
    float inv = 1.f;
    if constexpr (Q8) {
      uint32_t amax = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint32_t x[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
        for (int y = 0; y < 4; ++y) amax = max(amax, max(x[y] << 16 & 0x7fff0000u, x[y] & 0x7fff0000u));
      }
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // take the largest element's power of two out (|q'| < 2): f16 keeps every bit of a bf16 down to 2^-14 of
      // the row's largest, and below that an absolute 2^-25 of it
      const int e = min(max((int)(amax >> 23), 27), 227);
      inv = __int_as_float((254 - e) << 23);
      if (r < ROWS && part == 0) qscale[r] = __int_as_float(e << 23);
    }
    if (r < ROWS) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint32_t x[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int d = (part + i * 4) * 8 + 2 * y;                     // dims d, d + 1 of the row; word 0 or 1 of a B fragment
          const int t = Q8 ? d / (D / 4) : d % 8 / 2, kk = Q8 ? d % (D / 4) / 4 : d / 16, w = Q8 ? d % 4 / 2 : d % 16 / 8;
          const uint32_t h = Q8 ? pack2<FMT>(__uint_as_float(x[y] << 16) * inv, __uint_as_float(x[y] & 0xffff0000u) * inv) : x[y];
          reinterpret_cast<uint32_t*>(qs)[(((r >> 3) * MD + kk) * 32 + (r & 7) * 4 + t) * 2 + w] = h;
        }
      }
      masks[r * 4 + part] = mk;
    }
  }
  __syncthreads();

  // this thread's rows of n-tile n: 8 n + 2 tq, + 1
  float o[NT][MD][4], m[NT][2], l[NT][2], rf[NT][2];
  int er[NT][2];                                                        // 8-bit: exponent byte that the weights are relative to
  float top[NT][2];                                                     // and er + 12: beyond it a weight's exponent asks for another
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[n][h] = kNone;
      l[n][h] = 0.f;
      er[n][h] = 1;
      top[n][h] = 13.f;
      rf[n][h] = g.scale * 1.4426950408889634f * (Q8 ? qscale[8 * n + 2 * tq + h] * kHalfUnit<FMT> : 1.f);
#pragma unroll
      for (int d = 0; d < MD; ++d) o[n][d][h] = o[n][d][2 + h] = 0.f;
    }
  const uint2* qf = reinterpret_cast<const uint2*>(qs) + lane;
  int done = 0;                                                         // groups waited for
  bool ok = true, hit = false;
#pragma unroll 1
  for (int i = 0; i < my_groups; ++i) {
    const int s = i % NS;
    ok = __all_sync(0xffffffffu, mbar_wait(fb0 + s * 8, (i / NS) & 1, flags, g.spin));
    if (!ok) break;
    done = i + 1;
    const uint32_t kt = st0 + s * P::STAGE, vt = kt + HALF;
    const uint8_t* ks = stages + (warp * NS + s) * P::STAGE;
    const uint8_t* vs = ks + HALF;
    const uint8_t* ex = ex0 + s * 128;
    const int key0 = k_lo + (warp + 4 * i) * KG;
    const bool partial = key0 + KG > min(all_see, k_hi);                // some row does not see some key of the group
#pragma unroll 1
    for (int st = 0; st < KG / 16; ++st) {
      // ---- S^T of 16 keys: rows (keys) gq and gq + 8
      float sc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
      if constexpr (!Q8) {
#pragma unroll
        for (int kk = 0; kk < MD; ++kk) {
          const int key = st * 16 + (lane & 15), dim = kk * 16 + (lane >> 4) * 8;
          uint32_t a[4];
          ldsm_x4(kt + (dim >> 6) * KG * 128 + key * 128 + ((((dim & 63) >> 3) ^ (key & 7)) << 4), a);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint2 b = qf[(n * MD + kk) * 32];
            mma16816<FMT>(sc[n], a, b.x, b.y);
          }
        }
      } else {
#pragma unroll
        for (int u = 0; u < D / 64; ++u) {                              // 16 bytes of each key: four k-steps
          const int ch = tq * (D / 64) + u;
          uint4 w[2];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int key = st * 16 + gq + 8 * y;
            w[y] = *reinterpret_cast<const uint4*>(ks + key * D + ((D == 128 ? ch ^ (key & 7) : ch ^ ((key >> 1) & 3)) << 4));
          }
          const uint32_t w0[4] = {w[0].x, w[0].y, w[0].z, w[0].w}, w1[4] = {w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            uint32_t a[4];
            unpack4<FMT>(w0[y], a[0], a[2]);
            unpack4<FMT>(w1[y], a[1], a[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint2 b = qf[(n * MD + u * 4 + y) * 32];
              mma16816<FMT>(sc[n], a, b.x, b.y);
            }
          }
        }
      }
      // ---- scores in the log2 domain; masks
      float fv[2] = {1.f, 1.f}, ev[2] = {0.f, 0.f};                       // V's scale and its exponent byte (a NaN's counts as none)
      if constexpr (Q8) {
        const float fk0 = exp_scale(ex[st * 16 + gq]), fk1 = exp_scale(ex[st * 16 + gq + 8]);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int e = ex[64 + st * 16 + gq + 8 * y];
          fv[y] = exp_scale(e);
          ev[y] = e == 255 ? -INFINITY : (float)e;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            sc[n][h] *= rf[n][h] * fk0;
            sc[n][2 + h] *= rf[n][h] * fk1;
          }
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            sc[n][h] *= rf[n][h];
            sc[n][2 + h] *= rf[n][h];
          }
      }
      bool seen[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) seen[n][0] = seen[n][1] = seen[n][2] = seen[n][3] = true;
      if (partial) {
        const int left = k_hi - key0 - st * 16;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = 8 * n + 2 * tq + h;
            uint32_t see = sees32(g.mask ? masks + r * 4 : nullptr, 4, (r0 + min(r, nrows - 1)) / g.G, key0 + st * 16 - bi.ctx);
            if (left < 16) see &= left <= 0 ? 0u : (1u << left) - 1;
            seen[n][h] = see >> gq & 1;
            seen[n][2 + h] = see >> (gq + 8) & 1;
            if (!seen[n][h]) sc[n][h] = -INFINITY;
            if (!seen[n][2 + h]) sc[n][2 + h] = -INFINITY;
          }
      }
      // ---- a new reference where a score is more than 2^8 above it, or a weight with V's scale would pass 2^12 (in range of
      // f16).  A weight's exponent is the difference first: scores may be too large to hold V's exponent beside them.
      float x[NT][4];
      bool need = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          x[n][h] = sc[n][h] - m[n][h];
          x[n][2 + h] = sc[n][2 + h] - m[n][h];
          need = need || fmaxf(x[n][h], x[n][2 + h]) > 8.f || (Q8 && fmaxf(x[n][h] + ev[0], x[n][2 + h] + ev[1]) > top[n][h]);
        }
      if (__any_sync(0xffffffffu, need)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            auto row_max = [](float v) {
#pragma unroll
              for (int y = 4; y < 32; y <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, y));
              return v;
            };
            // (every lane takes part in every reduction: none of them behind a condition)
            const float mx = row_max(fmaxf(sc[n][h], sc[n][2 + h]));
            float tx = -INFINITY;
            if constexpr (Q8) tx = row_max(fmaxf(x[n][h] + ev[0], x[n][2 + h] + ev[1]));
            // a row moves by what it sees itself, whatever its neighbours in the tile see: the condition again, of the whole row
            const bool own = mx - m[n][h] > 8.f || (Q8 && tx > top[n][h]);
            const float mn = own ? fmaxf(m[n][h], mx) : m[n][h];
            const float df = m[n][h] - mn;
            float f = fast_exp2(df);
            l[n][h] *= f;
            x[n][h] = sc[n][h] - mn;
            x[n][2 + h] = sc[n][2 + h] - mn;
            if constexpr (Q8) {
              // relative to the largest weight x scale, which a V of a large scale and no weight does not raise.  Rounded down, so
              // that it does not creep up with every move of m; 1 .. 253 keep 2^(127 - er) a normal float.
              tx = row_max(fmaxf(x[n][h] + ev[0], x[n][2 + h] + ev[1]));
              const int en = own ? min(max((int)floorf(fmaxf(tx, df + (float)er[n][h])), 1), 253) : er[n][h];
              f = fast_exp2(df + (float)(er[n][h] - en));
              er[n][h] = en;
              top[n][h] = (float)(en + 12);
            }
            m[n][h] = mn;
#pragma unroll
            for (int d = 0; d < MD; ++d) {
              o[n][d][h] *= f;
              o[n][d][2 + h] *= f;
            }
          }
      }
      // ---- weights, and P^T as an operand
      uint32_t pb[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float w[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float p0 = fast_exp2(x[n][h]), p1 = fast_exp2(x[n][2 + h]);
          l[n][h] += p0 + p1;
          if constexpr (Q8) {
            const float rv = __int_as_float((254 - er[n][h]) << 23);    // 2^-(er - 127)
            w[h] = seen[n][h] ? p0 * fv[0] * rv : 0.f;
            w[2 + h] = seen[n][2 + h] ? p1 * fv[1] * rv : 0.f;
          } else {
            w[h] = p0;
            w[2 + h] = p1;
          }
        }
        pb[n][0] = transpose8(pack2<FMT>(w[0], w[1]));
        pb[n][1] = transpose8(pack2<FMT>(w[2], w[3]));
      }
      // ---- O^T += V^T P^T
      if constexpr (!Q8) {
#pragma unroll
        for (int d = 0; d < MD; ++d) {
          const int key = st * 16 + (lane & 7) + (lane >> 4) * 8, dim = d * 16 + ((lane >> 3) & 1) * 8;
          uint32_t a[4];
          ldsm_x4_t(vt + (dim >> 6) * KG * 128 + key * 128 + ((((dim & 63) >> 3) ^ (key & 7)) << 4), a);
          if (partial) {                 // 0 x NaN would reach every row: drop it here, put it back at the end
#pragma unroll
            for (int x = 0; x < 4; ++x) a[x] = drop_nonfinite(a[x], hit);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<FMT>(o[n][d], a, pb[n][0], pb[n][1]);
        }
      } else {
        // keys 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9 of this step, D / 8 bytes each
        uint32_t w[4][D / 32];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int key = st * 16 + 2 * tq + (x & 1) + (x >> 1) * 8;
          if constexpr (D == 128) {
            const uint4 v = *reinterpret_cast<const uint4*>(vs + key * D + ((gq ^ (key & 7)) << 4));
            w[x][0] = v.x, w[x][1] = v.y, w[x][2] = v.z, w[x][3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(vs + key * D + ((((gq >> 1) ^ ((key >> 1) & 3)) << 4) | (gq & 1) << 3));
            w[x][0] = v.x, w[x][1] = v.y;
          }
          if constexpr (FMT == EESD_KV_INT8)
#pragma unroll
            for (int y = 0; y < D / 32; ++y) w[x][y] ^= 0x80808080u;
        }
#pragma unroll
        for (int d = 0; d < MD; ++d) {
          uint32_t a[4];                                                // dims gq D/8 + 2 d (a0, a2) and + 1 (a1, a3)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int b = 2 * d + (x & 1), y = b >> 2, z = b & 3, k = x >> 1;
            if constexpr (FMT == EESD_KV_E4M3) {                        // bytes into the high halves of each lane
              a[x] = bytes_to_half2<FMT>(__byte_perm(w[2 * k][y], w[2 * k + 1][y], (4 + z) << 12 | z << 4));
            } else {
              a[x] = bytes_to_half2<FMT>(__byte_perm(__byte_perm(w[2 * k][y], w[2 * k + 1][y], (4 + z) << 4 | z), 0x64646464u, 0x4140));
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<FMT>(o[n][d], a, pb[n][0], pb[n][1]);
        }
      }
    }
    __syncwarp();                                                       // every lane is done with the stage
    if (lane == 0 && i + NS < my_groups) issue(i + NS);
  }
  if (!Q8 && hit) flags[1] = 1;
  if (!ok) {
    if (lane == 0) {
      set_status(g.status, kStatusTimeoutMma);
      flags[0] = 1;
      // groups issued and not waited for: one per stage at most
      const int issued = min(my_groups, done + NS);
      for (int i = done; i < issued; ++i) mbar_drain(fb0 + (i % NS) * 8, (i / NS) & 1);
    }
  }
  __syncthreads();
  if (flags[0]) return;

  // ---- the four warps' states, through the stage memory (every copy has landed)
  float* Ow = reinterpret_cast<float*>(stages);                         // [4][ROWS][OLD]
  float* Mw = Ow + 4 * ROWS * OLD;                                      // [4][ROWS] each: max, sum, eref
  float* Lw = Mw + 4 * ROWS;
  float* Ew = Lw + 4 * ROWS;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 8 * n + 2 * tq + h;
      float s = l[n][h];
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      if (gq == 0) {
        Mw[warp * ROWS + r] = m[n][h];
        Lw[warp * ROWS + r] = s;
        Ew[warp * ROWS + r] = (float)er[n][h];
      }
      float* dst = Ow + (warp * ROWS + r) * OLD;
#pragma unroll
      for (int d = 0; d < MD; ++d) {
        if constexpr (Q8) {
          *reinterpret_cast<float2*>(dst + gq * (D / 8) + 2 * d) = make_float2(o[n][d][h], o[n][d][2 + h]);
        } else {
          dst[d * 16 + gq] = o[n][d][h];
          dst[d * 16 + gq + 8] = o[n][d][2 + h];
        }
      }
    }
  __syncthreads();
  const bool whole = n_keys <= g.chunk;
  constexpr int LPR = D / 4;                                            // threads per row, 4 dims each
#pragma unroll 2
  for (int r = threadIdx.x / LPR; r < nrows; r += 128 / LPR) {
    const int d = threadIdx.x % LPR * 4;
    float M = kNone, top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      M = fmaxf(M, Mw[w * ROWS + r]);
    }
    if constexpr (Q8) {
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, Mw[w * ROWS + r] - M + Ew[w * ROWS + r]);
    }
    const float E = fminf(fmaxf(floorf(top), 1.f), 253.f);
    float L = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = fast_exp2(Mw[w * ROWS + r] - M);
      const float fo = Q8 ? fast_exp2(Mw[w * ROWS + r] - M + (Ew[w * ROWS + r] - E)) : f;
      L += f * Lw[w * ROWS + r];
      const float4 v = *reinterpret_cast<const float4*>(Ow + (w * ROWS + r) * OLD + d);
      acc[0] += fo * v.x, acc[1] += fo * v.y, acc[2] += fo * v.z, acc[3] += fo * v.w;
    }
    float inv = L == 0.f ? 0.f : 1.f / L;                               // a row that sees nothing: zeros
    const int R = r0 + r, node = R / g.G;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= inv;
    if constexpr (Q8) {                                                 // (the product of the three may pass fp32)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = acc[e] * kHalfUnit<FMT> * __int_as_float((int)E << 23);
    }
    if (!Q8 && flags[1]) {                                              // the dropped elements of keys this row sees
      const uint64_t* mk = g.mask ? masks + r * 4 : nullptr;
#pragma unroll 1
      for (int key = max(k_lo, min(all_see, k_hi) / KG * KG); key < k_hi; ++key)   // from the first partial group on
        if (sees32(mk, 4, node, key - bi.ctx) & 1) {
          const bf16* v = static_cast<const bf16*>(c.v) + ((size_t)slot0 + key) * D + d;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = __bfloat162float(v[e]);
            if (!(fabsf(x) < INFINITY)) acc[e] += x;
          }
        }
    }
    const size_t at = (size_t)(bi.start + node) * g.n_heads + kvh * g.G + R - node * g.G;
    if (whole) {
      *reinterpret_cast<uint2*>(out + at * D + d) = make_uint2(pack2<EESD_KV_MODEL>(acc[0], acc[1]), pack2<EESD_KV_MODEL>(acc[2], acc[3]));
    } else {
      const size_t p = at * g.splits + blockIdx.x;
      *reinterpret_cast<float4*>(g.part_o + p * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (d == 0) g.part_ml[p] = make_float2(M, L);
    }
  }
}

// Joins the key ranges of a row: partial outputs are normalised, range c weighs L_c 2^(M_c - M).  Ranges go round four
// classes (eight with D = 64, two to a warp) that are summed apart and then in order, without atomics: the same bits every time
// and with WPR = 1 or 4 warps per row.  Bound by the latency of its loads: 16 are in flight (a tree of 5
// nodes at 32 k slots over bf16, 42 ranges: 44 us in all, with four warps per row instead of one 2 us less; with the loads
// in one chain it was 52).
template <int D, int WPR>
__global__ void __launch_bounds__(128) attn_tree_join_kernel(TreeGeom g, CacheGeom c, int rows_per_tile, bf16* __restrict__ out) {
  pdl_trigger();
  pdl_wait();
  constexpr int GR = 128 / D, U = 4, CLS = 4 / WPR;                     // ranges of a warp's load, loads of a class in flight, classes of a warp
  __shared__ float4 part[4][33];                                        // WPR = 4: acc of the warps' lanes, and L
  BlockInfo bi;
  if (!load_block(g, c, blockIdx.z, bi)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = lane / (D / 4), kvh = blockIdx.y;
  const int R = WPR == 4 ? blockIdx.x : blockIdx.x * 4 + warp, cls0 = WPR == 4 ? warp : 0;
  if (R >= bi.T * g.G) return;
  const int node = R / g.G;
  // the key count of the row tile that R was in
  const int last = (min((R / rows_per_tile + 1) * rows_per_tile, bi.T * g.G) - 1) / g.G;
  const int n_keys = bi.ctx + (g.mask ? bi.T : last + 1);
  if (n_keys <= g.chunk) return;                                        // written whole
  const int n = (n_keys + g.chunk - 1) / g.chunk;
  const size_t at = (size_t)(bi.start + node) * g.n_heads + kvh * g.G + R % g.G;
  const float2* ml = g.part_ml + at * g.splits;
  const float4* po = reinterpret_cast<const float4*>(g.part_o + at * g.splits * D) + lane % (D / 4);
  float M = -INFINITY;
  for (int s = lane; s < n; s += 32) M = fmaxf(M, ml[s].x);
  M = warp_max(M);
  const float ms = M == -INFINITY ? 0.f : M;
  float L[CLS];
  float4 acc[CLS];
#pragma unroll
  for (int k = 0; k < CLS; ++k) L[k] = 0.f, acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < n; s0 += 4 * GR * U) {
    float4 v[U][CLS];
    float2 m[U][CLS];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < CLS; ++k) {
        const int s = min(s0 + (u * 4 + cls0 + k) * GR + grp, n - 1);
        m[u][k] = ml[s];
        v[u][k] = po[(size_t)s * (D / 4)];
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < CLS; ++k) {
        // a range that the row sees counts even where its weight vanishes: 0 x NaN is a NaN, as within a range
        if (s0 + (u * 4 + cls0 + k) * GR + grp >= n || m[u][k].y == 0.f) continue;
        const float w = m[u][k].y * fast_exp2(m[u][k].x - ms);
        L[k] += w;
        acc[k].x = fmaf(w, v[u][k].x, acc[k].x);
        acc[k].y = fmaf(w, v[u][k].y, acc[k].y);
        acc[k].z = fmaf(w, v[u][k].z, acc[k].z);
        acc[k].w = fmaf(w, v[u][k].w, acc[k].w);
      }
  }
  auto add = [](float4& a, const float4& b) { a.x += b.x, a.y += b.y, a.z += b.z, a.w += b.w; };
  if constexpr (GR == 2) {
#pragma unroll
    for (int k = 0; k < CLS; ++k) {
      L[k] += __shfl_xor_sync(0xffffffffu, L[k], 16);
      add(acc[k], make_float4(__shfl_xor_sync(0xffffffffu, acc[k].x, 16), __shfl_xor_sync(0xffffffffu, acc[k].y, 16),
                              __shfl_xor_sync(0xffffffffu, acc[k].z, 16), __shfl_xor_sync(0xffffffffu, acc[k].w, 16)));
    }
  }
  if constexpr (WPR == 4) {
    part[warp][lane] = acc[0];
    if (lane == 0) part[warp][32].x = L[0];
    __syncthreads();
    if (warp) return;
    for (int k = 1; k < 4; ++k) {
      add(acc[0], part[k][lane]);
      L[0] += part[k][32].x;
    }
  } else {
#pragma unroll
    for (int k = 1; k < CLS; ++k) {
      add(acc[0], acc[k]);
      L[0] += L[k];
    }
  }
  const float inv = L[0] == 0.f ? 0.f : 1.f / L[0];
  if (grp == 0)
    *reinterpret_cast<uint2*>(out + at * D + lane * 4) = make_uint2(pack2<EESD_KV_MODEL>(acc[0].x * inv, acc[0].y * inv),
                                                                    pack2<EESD_KV_MODEL>(acc[0].z * inv, acc[0].w * inv));
}

// ---------------------------------------------------------------- plan and launch
// One layer of the cache as a 2-D map of slots; box: `keys` slots of 64 bf16 (a 128-byte swizzled half row) or of
// the whole 8-bit row.
int encode_cache_map(CUtensorMap* map, const void* base, const EesdKvCache* c, int keys) {
  PFN_encodeTiled_t enc = tensor_map_encoder();
  if (!enc) return fail_arg(EESD_ERR_CUDA, "attn_tree: no tensor map encoder");
  const bool q8 = c->format != EESD_KV_MODEL;
  const int D = c->head_dim, eb = q8 ? 1 : 2;
  cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)c->max_batch * c->n_kv_heads * c->max_seq};
  cuuint64_t strides[1] = {(cuuint64_t)D * eb};
  cuuint32_t box[2] = {(cuuint32_t)(q8 ? D : 64), (cuuint32_t)keys};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(map, q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims,
                         strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         q8 && D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? EESD_OK : fail_arg(EESD_ERR_CUDA, "attn_tree: cache tensor map (%d)", (int)r);
}

constexpr int kWide = 8;   // from 9 key ranges on the join has four warps per row (42 ranges 46 -> 44 us; at 3 it would cost 50 -> 52)
struct Plan {
  bool tc;              // tcgen05 kernel (attn_tree_tc.cu), else mma.sync
  int nt;               // mma.sync: 8-row tiles per CTA
  int rows, tiles;      // rows per tile, row tiles of the largest block
  int chunk, splits;    // keys per CTA, key ranges of the longest row
  int ctas;             // tcgen05: persistent CTAs
  size_t ml_off, cuts_off, bytes;
};

int sm_count() {
  static const int n = [] {
    int dev = 0, v = 148;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) v = 148;
    return v;
  }();
  return n;
}

Plan plan_for(const EesdKvCache* c, const EesdTree* t, int n_heads, int split_keys) {
  Plan p{};
  const int G = n_heads / c->n_kv_heads, rows = t->max_nodes * G;
  // Up to 32 rows the mma.sync kernel, whose cost grows with the rows in steps of 8; beyond, the tcgen05 kernel, whose tiles
  // have 128 rows whatever is in them.  With 32 rows (mma.sync / tcgen05): 64 blocks at 129 to 1023 slots over bf16 41 / 59 us,
  // over int8 50 / 87; 16 blocks at 300 to 4000 slots 53 / 42 and 66 / 52.  With 36 rows: 68 / 60, 86 / 89, 81 / 42, 103 / 52.
  p.tc = rows > 32;
  p.nt = std::min(4, (rows + 7) / 8);
  p.rows = p.tc ? (rows <= 128 ? 128 : 256) : 8 * p.nt;
  p.tiles = (rows + p.rows - 1) / p.rows;
  const long long units = (long long)t->n_blocks * c->n_kv_heads * p.tiles;
  p.chunk = split_keys;
  size_t parts = 0;     // partial rows
  if (p.tc) {
    // a CTA for every unit, and more where runs of 8 tiles and more remain
    const long long most = units * ((t->max_ctx + 63) / 64);
    p.ctas = (int)std::max(1LL, std::min<long long>(sm_count(), std::max(units, (most + 7) / 8)));
    if (!p.chunk) parts = (size_t)p.ctas * 2 * p.rows;
  } else if (!p.chunk) {
    const int slots = sm_count() * (p.nt == 4 || (p.nt == 3 && c->head_dim == 128 && c->format != EESD_KV_MODEL) ? 2 : 3);
    const int want = (int)std::max(1LL, slots / std::max(1LL, units));
    const int per = (t->max_ctx + want - 1) / want;
    // up to 512 slots the join costs more than a second range saves (one token at 300 slots 8.3 us whole, 10.5 in two; 8 at
    // 500: 14 and 17); at 1000 it no longer does (in two 17, in four 15)
    p.chunk = t->max_ctx <= 512 ? 512 : (per + 255) / 256 * 256;
  }
  p.splits = p.chunk ? (t->max_ctx + p.chunk - 1) / p.chunk : 1;
  if (p.splits > 1) parts = (size_t)t->n_tokens * n_heads * p.splits;
  const auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  p.ml_off = up(parts * c->head_dim * 4);
  p.cuts_off = p.ml_off + up(parts * 8);
  p.bytes = std::max<size_t>(p.cuts_off + (p.tc ? up((size_t)p.ctas * sizeof(TcCut)) : 0), 256);
  return p;
}

template <int D, int FMT, int NT>
cudaError_t launch_mma(const Plan& p, const TreeGeom& g, const CacheGeom& c, const CUtensorMap& km, const CUtensorMap& vm, int n_blocks,
                       const void* q, void* out, cudaStream_t s) {
  using S = MmaShape<D, FMT, NT>;
  auto kernel = attn_tree_mma_kernel<D, FMT, NT>;
  static SmemOnce once;
  const cudaError_t e = once.set(reinterpret_cast<const void*>(kernel), S::smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(kernel, dim3(p.splits, p.tiles * c.n_kv_heads, n_blocks), dim3(128), S::smem, s, km, vm, g, c,
                    static_cast<const bf16*>(q), static_cast<bf16*>(out));
}
template <int D, int FMT>
cudaError_t launch_nt(const Plan& p, const TreeGeom& g, const CacheGeom& c, const CUtensorMap& km, const CUtensorMap& vm, int nb,
                      const void* q, void* out, cudaStream_t s) {
  switch (p.nt) {
    case 1: return launch_mma<D, FMT, 1>(p, g, c, km, vm, nb, q, out, s);
    case 2: return launch_mma<D, FMT, 2>(p, g, c, km, vm, nb, q, out, s);
    case 3: return launch_mma<D, FMT, 3>(p, g, c, km, vm, nb, q, out, s);
    default: return launch_mma<D, FMT, 4>(p, g, c, km, vm, nb, q, out, s);
  }
}

template <typename T, int FMT, int D>
cudaError_t launch_simt(const TreeGeom& g, const CacheGeom& c, int n_blocks, const void* q, void* out, cudaStream_t s) {
  const dim3 grid((g.max_nodes * g.G + 31) / 32, c.n_kv_heads, n_blocks);
  constexpr size_t smem = (32 * D + 32 * (D + 1) + 32 * D) * 4;
  static SmemOnce once;
  const cudaError_t e = once.set(reinterpret_cast<const void*>(attn_tree_simt_kernel<T, FMT, D>), smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(attn_tree_simt_kernel<T, FMT, D>, grid, dim3(128), smem, s, g, c, static_cast<const T*>(q), static_cast<T*>(out));
}
cudaError_t launch_f32(int fmt, int D, const TreeGeom& g, const CacheGeom& c, int nb, const void* q, void* out, cudaStream_t s) {
  switch (fmt * 2 + (D == 128)) {
    case 0: return launch_simt<float, EESD_KV_MODEL, 64>(g, c, nb, q, out, s);
    case 1: return launch_simt<float, EESD_KV_MODEL, 128>(g, c, nb, q, out, s);
    case 2: return launch_simt<float, EESD_KV_E4M3, 64>(g, c, nb, q, out, s);
    case 3: return launch_simt<float, EESD_KV_E4M3, 128>(g, c, nb, q, out, s);
    case 4: return launch_simt<float, EESD_KV_INT8, 64>(g, c, nb, q, out, s);
    default: return launch_simt<float, EESD_KV_INT8, 128>(g, c, nb, q, out, s);
  }
}
cudaError_t launch_bf16(int fmt, int D, const Plan& p, const TreeGeom& g, const CacheGeom& c, const CUtensorMap& km, const CUtensorMap& vm,
                        int nb, const void* q, void* out, cudaStream_t s) {
  switch (fmt * 2 + (D == 128)) {
    case 0: return launch_nt<64, EESD_KV_MODEL>(p, g, c, km, vm, nb, q, out, s);
    case 1: return launch_nt<128, EESD_KV_MODEL>(p, g, c, km, vm, nb, q, out, s);
    case 2: return launch_nt<64, EESD_KV_E4M3>(p, g, c, km, vm, nb, q, out, s);
    case 3: return launch_nt<128, EESD_KV_E4M3>(p, g, c, km, vm, nb, q, out, s);
    case 4: return launch_nt<64, EESD_KV_INT8>(p, g, c, km, vm, nb, q, out, s);
    default: return launch_nt<128, EESD_KV_INT8>(p, g, c, km, vm, nb, q, out, s);
  }
}

int check_attn(int dtype, const EesdKvCache* c, int layer, const EesdTree* t, int n_heads, int split_keys) {
  int rc = check_cache("attn_tree", dtype, c, layer);
  if (!rc) rc = check_tree("attn_tree", t);
  if (rc) return rc;
  if (n_heads <= 0 || n_heads % c->n_kv_heads) return fail_arg(EESD_ERR_ARG, "attn_tree: heads %d / %d", n_heads, c->n_kv_heads);
  if (split_keys < 0 || split_keys % 256) return fail_arg(EESD_ERR_ARG, "attn_tree: split_keys %d (0 or a multiple of 256)", split_keys);
  const long long rows = (long long)t->max_nodes * (n_heads / c->n_kv_heads);   // the grids and the schedule count them in 32 bits
  if (rows > 1 << 24 || rows * t->n_blocks >= 1LL << 37)
    return fail_arg(EESD_ERR_ARG, "attn_tree: %d blocks of max_nodes %d x %d heads are too many rows", t->n_blocks, t->max_nodes,
                    n_heads / c->n_kv_heads);
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
  if (dtype == EESD_F32 || t->n_tokens == 0 || t->n_blocks == 0) return 256;
  return plan_for(c, t, n_heads, split_keys).bytes;
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
  TreeGeom g{n_heads, n_heads / c->n_kv_heads, t->n_tokens, t->max_nodes, t->max_ctx, t->words, t->blk, t->mask, ld_q,
             1.f / sqrtf((float)c->head_dim), status, spin_limit(), 0, 0, false, nullptr, nullptr};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == EESD_F32) {
    e = launch_f32(c->format, c->head_dim, g, cg, t->n_blocks, q, out, s);
  } else {
    const Plan p = plan_for(c, t, n_heads, split_keys);
    g.chunk = p.chunk;
    g.splits = p.splits;
    g.part_o = static_cast<float*>(workspace);
    g.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + p.ml_off);
    const int keys = p.tc ? 64 : 4096 / (c->head_dim * (c->format == EESD_KV_MODEL ? 2 : 1));
    CUtensorMap km, vm;
    if ((rc = encode_cache_map(&km, cg.k, c, keys)) || (rc = encode_cache_map(&vm, cg.v, c, keys))) return rc;
    if (p.tc) {
      const TcSchedule sc{p.ctas, p.rows, p.tiles, t->n_blocks * p.tiles, split_keys / 64,
                          reinterpret_cast<TcCut*>(static_cast<uint8_t*>(workspace) + p.cuts_off)};
      e = launch_attn_tree_tc(c->format, c->head_dim, sc, g, cg, km, vm, q, out, s);
    } else {
      g.sort = t->n_blocks > 1 && t->n_blocks <= kSorted && (long long)t->n_blocks * c->n_kv_heads * p.tiles * p.splits > sm_count();
      e = launch_bf16(c->format, c->head_dim, p, g, cg, km, vm, t->n_blocks, q, out, s);
    }
    if (e == cudaSuccess && p.splits > 1) {
      // four warps per row where a row may be in many ranges
      const bool wide = p.splits > kWide;
      const int rows = t->max_nodes * g.G;
      const dim3 grid(wide ? rows : (rows + 3) / 4, c->n_kv_heads, t->n_blocks);
      auto kernel = c->head_dim == 64 ? (wide ? attn_tree_join_kernel<64, 4> : attn_tree_join_kernel<64, 1>)
                                      : (wide ? attn_tree_join_kernel<128, 4> : attn_tree_join_kernel<128, 1>);
      e = launch_pdl(kernel, grid, dim3(128), 0, s, g, cg, p.rows, static_cast<bf16*>(out));
    }
  }
  return e == cudaSuccess ? EESD_OK : fail_arg(EESD_ERR_CUDA, "attn_tree: launch: %s", cudaGetErrorString(e));
}

}  // extern "C"
