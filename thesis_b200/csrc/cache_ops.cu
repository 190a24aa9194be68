// Tree metadata, quantising KV append and read-back, tree acceptance and cache compaction: the kernels
// around the tree attention, and their C entry points.
#include <stdarg.h>
#include <stdio.h>

#include "attn_tree.h"
#include "cache.cuh"
#include "kernels.h"

namespace eesd {

int fail_arg(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return code;
}

int check_stream(const char* who, void* stream) {
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  cudaError_t e = cudaStreamIsCapturing(s, &cap);
  if (e == cudaSuccess && cap != cudaStreamCaptureStatusNone) return EESD_OK;   // the device query below would end the capture
  int dev = -1, sdev = -2;
  if (e == cudaSuccess) e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaStreamGetDevice(s, &sdev);
  if (e != cudaSuccess) return fail_arg(EESD_ERR_CUDA, "%s: stream: %s", who, cudaGetErrorString(e));
  if (dev != sdev) return fail_arg(EESD_ERR_ARG, "%s: the stream belongs to device %d, the current device is %d", who, sdev, dev);
  return EESD_OK;
}

int check_cache(const char* who, int dtype, const EesdKvCache* c, int layer) {
  if (!c || !c->k || !c->v) return fail_arg(EESD_ERR_ARG, "%s: null cache", who);
  if (dtype != EESD_BF16 && dtype != EESD_F32) return fail_arg(EESD_ERR_ARG, "%s: dtype %d", who, dtype);
  if (c->format < EESD_KV_MODEL || c->format > EESD_KV_INT8) return fail_arg(EESD_ERR_ARG, "%s: cache format %d", who, c->format);
  if (c->head_dim != 64 && c->head_dim != 128) return fail_arg(EESD_ERR_ARG, "%s: head_dim %d (64 or 128)", who, c->head_dim);
  if (c->n_layers <= 0 || c->max_batch <= 0 || c->n_kv_heads <= 0 || c->max_seq <= 0 || c->max_seq % 16)
    return fail_arg(EESD_ERR_ARG, "%s: cache sizes (max_seq must be a multiple of 16)", who);
  if ((long long)c->max_batch * c->n_kv_heads * c->max_seq >= (1LL << 31))
    return fail_arg(EESD_ERR_ARG, "%s: more than 2^31 slots in one layer of the cache", who);
  if (layer < 0 || layer >= c->n_layers) return fail_arg(EESD_ERR_ARG, "%s: layer %d of %d", who, layer, c->n_layers);
  uintptr_t a = reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v);
  if (c->format != EESD_KV_MODEL) {
    if (!c->k_exp || !c->v_exp) return fail_arg(EESD_ERR_ARG, "%s: an 8-bit cache needs k_exp and v_exp", who);
    a |= reinterpret_cast<uintptr_t>(c->k_exp) | reinterpret_cast<uintptr_t>(c->v_exp);
  }
  if (a & 15) return fail_arg(EESD_ERR_ARG, "%s: cache pointers must be 16-byte aligned", who);
  return EESD_OK;
}

int check_tree(const char* who, const EesdTree* t) {
  if (!t) return fail_arg(EESD_ERR_ARG, "%s: null tree", who);
  if (t->n_tokens < 0 || t->n_blocks < 0 || t->n_blocks > 65535)
    return fail_arg(EESD_ERR_ARG, "%s: n_tokens %d, n_blocks %d (at most 65535)", who, t->n_tokens, t->n_blocks);
  if (t->n_tokens == 0 || t->n_blocks == 0) return EESD_OK;
  if (!t->blk || t->max_nodes <= 0 || t->max_ctx <= 0) return fail_arg(EESD_ERR_ARG, "%s: missing block metadata", who);
  if (t->mask && (t->max_nodes > EESD_TREE_MAX_NODES || t->words != (t->max_nodes + 63) / 64))
    return fail_arg(EESD_ERR_ARG, "%s: a mask needs max_nodes <= %d and words = (max_nodes + 63) / 64", who, EESD_TREE_MAX_NODES);
  return EESD_OK;
}

CacheGeom cache_layer(const EesdKvCache* c, int dtype, int layer) {
  const size_t slots = (size_t)c->max_batch * c->n_kv_heads * c->max_seq * layer;
  const size_t eb = cache_elem_bytes(c, dtype);
  CacheGeom g{c->n_kv_heads, c->max_batch, c->max_seq, nullptr, nullptr, nullptr, nullptr};
  g.k = static_cast<const uint8_t*>(c->k) + slots * c->head_dim * eb;
  g.v = static_cast<const uint8_t*>(c->v) + slots * c->head_dim * eb;
  if (c->format != EESD_KV_MODEL) {
    g.ke = c->k_exp + slots;
    g.ve = c->v_exp + slots;
  }
  return g;
}

namespace {

// ---------------------------------------------------------------- metadata
// One CTA per block.  Each thread walks up from its nodes through the parents in shared memory (at most
// depth steps), counting the depth and setting the ancestors' bits.  Latency-bound: 4 to 5 us for 64 trees of 5 nodes (profiled).
// Tokens that no block covers get -1, or they would keep what an earlier round left there and be written to its slots.  A block
// followed by the next one, as usual, has nothing to do for that; else its CTA looks for the block that comes next.
__global__ void __launch_bounds__(128) tree_meta_kernel(EesdTree t, int max_batch, int max_seq, int* status) {
  pdl_trigger();
  pdl_wait();
  __shared__ int16_t par[EESD_TREE_MAX_NODES];
  const int b = blockIdx.x;
  const int start = t.blk[4 * b], T = t.blk[4 * b + 1], row = t.blk[4 * b + 2], ctx = t.blk[4 * b + 3];
  auto fits = [&](int s, int n) { return s >= 0 && n > 0 && s <= t.n_tokens - n; };
  __shared__ int next;
  auto uncovered = [&](int from) {                                      // tokens from `from` up to the next block
    __syncthreads();
    if (threadIdx.x == 0) next = t.n_tokens;
    __syncthreads();
    for (int j = threadIdx.x; j < t.n_blocks; j += blockDim.x) {
      const int s = t.blk[4 * j], n = t.blk[4 * j + 1];
      if (fits(s, n) && s + n > from) atomicMin(&next, max(s, from));
    }
    __syncthreads();
    for (int i = from + threadIdx.x; i < next; i += blockDim.x) t.tok_pos[i] = t.tok_slot[i] = t.tok_row[i] = -1;
  };
  if (b == 0 && !(start == 0 && fits(start, T))) uncovered(0);
  if (!fits(start, T)) {
    if (threadIdx.x == 0) set_status(status, kStatusBadIndex);
    return;
  }
  const int end = start + T;
  if (end < t.n_tokens && !(b + 1 < t.n_blocks && t.blk[4 * b + 4] == end && fits(end, t.blk[4 * b + 5]))) uncovered(end);
  const bool ok = row >= 0 && row < max_batch && ctx >= 0 && T <= t.max_nodes && ctx <= max_seq - T;
  if (!ok && threadIdx.x == 0) set_status(status, kStatusBadIndex);
  const bool tree = t.parent && T <= EESD_TREE_MAX_NODES;   // the entry point refuses parents with larger max_nodes
  if (tree)
    for (int i = threadIdx.x; i < T; i += blockDim.x) {
      int p = t.parent[start + i];
      if (p < -1 || p >= i) {
        set_status(status, kStatusBadIndex);
        p = -1;
      }
      par[i] = (int16_t)p;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < T; i += blockDim.x) {
    uint64_t m0 = 0, m1 = 0, m2 = 0, m3 = 0;
    int depth = -1;
    if (tree) {
      for (int j = i; j >= 0; j = par[j]) {
        ++depth;
        const uint64_t bit = 1ull << (j & 63);
        m0 |= (j >> 6) == 0 ? bit : 0;
        m1 |= (j >> 6) == 1 ? bit : 0;
        m2 |= (j >> 6) == 2 ? bit : 0;
        m3 |= (j >> 6) == 3 ? bit : 0;
      }
    } else {
      depth = i;
      auto upto = [&](int w) { return i >= 64 * w + 63 ? ~0ull : i < 64 * w ? 0ull : (2ull << (i - 64 * w)) - 1; };
      m0 = upto(0);
      m1 = upto(1);
      m2 = upto(2);
      m3 = upto(3);
    }
    const int tok = start + i;
    t.tok_pos[tok] = ok ? ctx + depth : -1;
    t.tok_slot[tok] = ok ? ctx + i : -1;
    t.tok_row[tok] = ok ? row : -1;
    if (t.mask) {
      uint64_t* m = t.mask + (size_t)tok * t.words;
      m[0] = m0;
      if (t.words > 1) m[1] = m1;
      if (t.words > 2) m[2] = m2;
      if (t.words > 3) m[3] = m3;
    }
  }
}

// ---------------------------------------------------------------- append
// 4 consecutive elements as floats
template <typename T> __device__ __forceinline__ void load4(const T* p, float (&x)[4]);
template <> __device__ __forceinline__ void load4<float>(const float* p, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
template <> __device__ __forceinline__ void load4<bf16>(const bf16* p, float (&x)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
  x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
}
// 8 elements, written once and read by others: past the caches
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
    __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(x[4], x[5], x[6], x[7]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 a = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&a);
    }
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// Four consecutive elements of each half of a head, that is four rotation pairs, and the tables' entries for them.  The
// roundings are those of the reference's apply_rope in the model dtype: every product and every sum rounded, no contraction.
template <typename T> struct Rope;
template <> struct Rope<float> {
  using Quad = float4;
  float4 c1, c2, s1, s2;
  __device__ void load(const float* cosb, const float* sinb, int half) {
    c1 = *reinterpret_cast<const float4*>(cosb), c2 = *reinterpret_cast<const float4*>(cosb + half);
    s1 = *reinterpret_cast<const float4*>(sinb), s2 = *reinterpret_cast<const float4*>(sinb + half);
  }
  static __device__ void turn(float& x, float& y, float c1, float c2, float s1, float s2) {
    const float a = __fadd_rn(__fmul_rn(x, c1), __fmul_rn(-y, s1)), b = __fadd_rn(__fmul_rn(y, c2), __fmul_rn(x, s2));
    x = a, y = b;
  }
  __device__ void rotate(float4& x, float4& y) const {
    turn(x.x, y.x, c1.x, c2.x, s1.x, s2.x);
    turn(x.y, y.y, c1.y, c2.y, s1.y, s2.y);
    turn(x.z, y.z, c1.z, c2.z, s1.z, s2.z);
    turn(x.w, y.w, c1.w, c2.w, s1.w, s2.w);
  }
  static __device__ uint32_t amax(const float4& x, const float4& y) {   // bits of the largest |element| as fp32
    auto m = [](const float4& v) {
      return max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu),
                 max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
    };
    return max(m(x), m(y));
  }
  static __device__ float4 floats(const float4& x) { return x; }
};
// bf16: two elements an instruction.  A product of two bf16 is exact in fp32, and so is a sum of two as far as bf16 can
// tell, so rounding once to bf16 is what rounding the fp32 result is.
template <> struct Rope<bf16> {
  using Quad = uint2;
  uint2 c1, c2, s1, s2;
  static __device__ uint2 rounded(const float* p) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
  __device__ void load(const float* cosb, const float* sinb, int half) {
    c1 = rounded(cosb), c2 = rounded(cosb + half), s1 = rounded(sinb), s2 = rounded(sinb + half);
  }
  static __device__ void turn(uint32_t& x, uint32_t& y, uint32_t c1, uint32_t c2, uint32_t s1, uint32_t s2) {
    auto v = [](const uint32_t& u) { return *reinterpret_cast<const __nv_bfloat162*>(&u); };
    const __nv_bfloat162 a = __hsub2_rn(__hmul2_rn(v(x), v(c1)), __hmul2_rn(v(y), v(s1)));
    const __nv_bfloat162 b = __hadd2_rn(__hmul2_rn(v(y), v(c2)), __hmul2_rn(v(x), v(s2)));
    x = *reinterpret_cast<const uint32_t*>(&a), y = *reinterpret_cast<const uint32_t*>(&b);
  }
  __device__ void rotate(uint2& x, uint2& y) const {
    turn(x.x, y.x, c1.x, c2.x, s1.x, s2.x);
    turn(x.y, y.y, c1.y, c2.y, s1.y, s2.y);
  }
  static __device__ uint32_t amax(const uint2& x, const uint2& y) {
    const uint32_t m = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(y.x & 0x7fff7fffu, y.y & 0x7fff7fffu));
    return max(m << 16, m & 0xffff0000u);
  }
  static __device__ float4 floats(const uint2& x) {
    return make_float4(__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u), __uint_as_float(x.y << 16),
                       __uint_as_float(x.y & 0xffff0000u));
  }
};

// A group of D / 8 lanes owns one head of one token: lane l holds elements 4 l .. 4 l + 3 of both halves,
// that is four rotation pairs, so the rotation needs no exchange and the largest |x| of the vector is a
// shuffle over the group.  Bound by the bytes of qkv, q_out and the cache, at few tokens by the chain of loads: a thread's
// kBatch heads are asked for before the token's position, on which the tables and the slot hang, is there.  Append and
// read-back of 320 tokens (32 query and 8 KV heads of 128, e4m3) take 6.1 us of device time, of 2048 tokens over int8 15.5 us,
// 3.8 TB/s (19 with the rotation of bf16 in fp32).
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(256) kv_append_kernel(const T* qkv, int ld_qkv, T* q_out, int ld_qo,
                                                        int n_heads, const int32_t* __restrict__ tok_pos,
                                                        const int32_t* __restrict__ tok_slot,
                                                        const int32_t* __restrict__ tok_row, CacheGeom c,
                                                        const float* __restrict__ cosb, const float* __restrict__ sinb,
                                                        int rope_len, int* status) {
  pdl_trigger();
  pdl_wait();
  constexpr int L = D / 8, GROUPS = 256 / L, H2 = D / 2, kBatch = 3;
  const int t = blockIdx.x, l = threadIdx.x % L, first = threadIdx.x / L;
  const T* base = qkv + (size_t)t * ld_qkv + 4 * l;
  const int heads = n_heads + 2 * c.n_kv_heads;
  using R = Rope<T>;
  typename R::Quad x[kBatch][2];
  // every lane of a warp takes part in the shuffles: head numbers past the end repeat the last head, unstored
  auto load = [&](int h0) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = min(h0 + b * GROUPS, heads - 1);
      x[b][0] = *reinterpret_cast<const typename R::Quad*>(base + (size_t)h * D);
      x[b][1] = *reinterpret_cast<const typename R::Quad*>(base + (size_t)h * D + H2);
    }
  };
  load(first);
  const int pos = tok_pos[t], row = tok_row[t], slot = tok_slot[t];
  if (pos < 0 || pos >= rope_len || row < 0 || row >= c.max_batch || slot < 0 || slot >= c.max_seq) {
    if (threadIdx.x == 0 && (pos != -1 || row != -1 || slot != -1)) set_status(status, kStatusBadIndex);   // all -1: padding
    return;
  }
  R rope;
  rope.load(cosb + (size_t)pos * D + 4 * l, sinb + (size_t)pos * D + 4 * l, H2);
  for (int h0 = first;; load(h0)) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int hh = h0 + b * GROUPS;
      const bool in = hh < heads;
      const int h = in ? hh : heads - 1;
      typename R::Quad &x1 = x[b][0], &x2 = x[b][1];
      if (h < n_heads + c.n_kv_heads) rope.rotate(x1, x2);
      if (h < n_heads) {
        if (in) {
          T* q = q_out + (size_t)t * ld_qo + (size_t)h * D + 4 * l;
          *reinterpret_cast<typename R::Quad*>(q) = x1;
          *reinterpret_cast<typename R::Quad*>(q + H2) = x2;
        }
        if constexpr (FMT == EESD_KV_MODEL) continue;
      }
      const bool isk = h < n_heads + c.n_kv_heads;
      const size_t at = cache_slot(c, row, isk ? h - n_heads : h - n_heads - c.n_kv_heads, slot);
      if constexpr (FMT == EESD_KV_MODEL) {
        if (in) {
          T* d = static_cast<T*>(const_cast<void*>(isk ? c.k : c.v)) + at * D + 4 * l;
          *reinterpret_cast<typename R::Quad*>(d) = x1;
          *reinterpret_cast<typename R::Quad*>(d + H2) = x2;
        }
      } else {
        uint32_t amax = R::amax(x1, x2);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (!in || h < n_heads) continue;
        const int eb = exp_byte<FMT>(amax);
        const float inv = exp_inv_scale(eb);
        uint32_t w1 = 0, w2 = 0;
        if (eb != 255) {
          const float4 y1 = R::floats(x1), y2 = R::floats(x2);
          w1 = quant2<FMT>(y1.x * inv, y1.y * inv) | quant2<FMT>(y1.z * inv, y1.w * inv) << 16;
          w2 = quant2<FMT>(y2.x * inv, y2.y * inv) | quant2<FMT>(y2.z * inv, y2.w * inv) << 16;
        }
        uint8_t* d = static_cast<uint8_t*>(const_cast<void*>(isk ? c.k : c.v)) + at * D + 4 * l;
        *reinterpret_cast<uint32_t*>(d) = w1;
        *reinterpret_cast<uint32_t*>(d + H2) = w2;
        if (l == 0) const_cast<uint8_t*>(isk ? c.ke : c.ve)[at] = (uint8_t)eb;
      }
    }
    h0 += kBatch * GROUPS;
    if (h0 - first >= heads) break;
  }
}

// ---------------------------------------------------------------- read-back
// A warp per token, neighbouring lanes on neighbouring 8-element chunks of a head (an 8-byte load in the 8-bit formats,
// 16-byte stores), four loads of different heads in flight.  Bound by the bytes of the output: contexts of 64 requests (129 to 1023 slots,
// 8 KV heads of 128, int8) take 39 us, 91 % of the copy rate (a thread per 8 elements with a 64-bit division: 52 us).
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(256) kv_read_kernel(CacheGeom c, const int32_t* __restrict__ tok_slot,
                                                      const int32_t* __restrict__ tok_row, int n_tok, T* __restrict__ k_out,
                                                      T* __restrict__ v_out, int* status) {
  pdl_trigger();
  pdl_wait();
  constexpr int C = D / 8, STEP = 32 / C, U = 4;
  const bool isk = blockIdx.y == 0 && k_out;
  T* out = isk ? k_out : v_out;
  const void* src = isk ? c.k : c.v;
  const uint8_t* exps = isk ? c.ke : c.ve;
  const int lane = threadIdx.x & 31, ch = lane % C;
  for (long long t = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); t < n_tok; t += (long long)gridDim.x * 8) {
    const int row = tok_row[t], slot = tok_slot[t];
    if (row < 0 || row >= c.max_batch || slot < 0 || slot >= c.max_seq) {
      if (row != -1 || slot != -1) set_status(status, kStatusBadIndex);   // both -1: padding
      continue;
    }
    for (int h0 = lane / C; h0 < c.n_kv_heads; h0 += U * STEP) {
      float x[U][8];
      uint2 w[U];
      int e[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h0 + u * STEP;
        if (h >= c.n_kv_heads) break;
        const size_t at = cache_slot(c, row, h, slot);
        if constexpr (FMT == EESD_KV_MODEL) {
          load4<T>(static_cast<const T*>(src) + at * D + ch * 8, *reinterpret_cast<float(*)[4]>(x[u]));
          load4<T>(static_cast<const T*>(src) + at * D + ch * 8 + 4, *reinterpret_cast<float(*)[4]>(x[u] + 4));
        } else {
          w[u] = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(src) + at * D + ch * 8);
          e[u] = exps[at];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h0 + u * STEP;
        if (h >= c.n_kv_heads) break;
        if constexpr (FMT != EESD_KV_MODEL) {
          const float s = exp_scale(e[u]) * kHalfUnit<FMT>;
          uint32_t p[4];
          unpack4<FMT>(w[u].x, p[0], p[1]);
          unpack4<FMT>(w[u].y, p[2], p[3]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = half2_to_float2(p[i]);
            x[u][2 * i] = f.x * s, x[u][2 * i + 1] = f.y * s;
          }
        }
        store8<T>(out + ((size_t)t * c.n_kv_heads + h) * D + ch * 8, x[u]);
      }
    }
  }
}

// ---------------------------------------------------------------- acceptance
// One warp per block: the walk is serial, each step one vote over the nodes behind the current one.  With the
// compaction 5.0 us of device time for 4 trees of 15 nodes, 8.8 us for 32 of 31.
__global__ void __launch_bounds__(32) tree_accept_kernel(EesdTree t, const int32_t* __restrict__ y,
                                                         const int32_t* __restrict__ ids, int32_t* __restrict__ path,
                                                         int32_t* __restrict__ n_acc, int32_t* __restrict__ next, int* status) {
  pdl_trigger();
  pdl_wait();
  __shared__ int32_t par[EESD_TREE_MAX_NODES], id[EESD_TREE_MAX_NODES], ys[EESD_TREE_MAX_NODES];
  const int b = blockIdx.x, lane = threadIdx.x;
  const int start = t.blk[4 * b], T = t.blk[4 * b + 1];
  int32_t* out = path + (size_t)b * t.max_nodes;
  bool ok = start >= 0 && T > 0 && T <= t.max_nodes && T <= EESD_TREE_MAX_NODES && start <= t.n_tokens - T;
  if (ok) {
    for (int i = lane; i < T; i += 32) {
      par[i] = t.parent ? t.parent[start + i] : i - 1;
      id[i] = ids[start + i];
      ys[i] = y[start + i];
    }
    __syncwarp();
  } else if (lane == 0) {
    set_status(status, kStatusBadIndex);
  }
  int cur = 0, len = 0;
  if (ok) {
    for (;;) {
      if (lane == 0) out[len] = cur;
      ++len;
      const int want = ys[cur];
      int child = -1;
      // children come after their parent, so the walk ends after at most T nodes
      for (int i0 = (cur + 1) & ~31; i0 < T && child < 0; i0 += 32) {
        const int i = i0 + lane;
        const unsigned hit = __ballot_sync(0xffffffffu, i > cur && i < T && par[i] == cur && id[i] == want);
        if (hit) child = i0 + __ffs(hit) - 1;
      }
      if (child < 0) break;
      cur = child;
    }
  }
  for (int i = len + lane; i < t.max_nodes; i += 32) out[i] = -1;
  if (lane == 0) {
    n_acc[b] = len - 1;
    next[b] = ok ? ys[cur] : -1;
  }
}

// ---------------------------------------------------------------- compaction
// grid (16-byte chunks of all layers, heads, K and V; blocks).  A thread owns one 16-byte column of one
// (layer, head) and moves its path slots in rising order: path[j] >= j, so every source is read before the
// move that overwrites it (four loads, then four stores).  Latency-bound: few bytes over many threads.
__global__ void __launch_bounds__(256) kv_compact_kernel(uint8_t* __restrict__ k, uint8_t* __restrict__ v,
                                                         uint8_t* __restrict__ ke, uint8_t* __restrict__ ve, int n_layers,
                                                         int n_kv_heads, int max_batch, int max_seq, int slot_bytes, EesdTree t,
                                                         const int32_t* __restrict__ path,
                                                         const int32_t* __restrict__ n_acc, int* status) {
  pdl_trigger();
  pdl_wait();
  __shared__ int16_t src[EESD_TREE_MAX_NODES];
  __shared__ int first;
  const int b = blockIdx.y;
  const int T = t.blk[4 * b + 1], row = t.blk[4 * b + 2], ctx = t.blk[4 * b + 3], acc = n_acc[b];
  bool ok = T > 0 && T <= t.max_nodes && T <= EESD_TREE_MAX_NODES && row >= 0 && row < max_batch && ctx >= 0 && ctx <= max_seq - T &&
            acc >= 0 && acc < T;
  if (threadIdx.x == 0) first = acc + 1;
  __syncthreads();
  // another block on slots of this one would read what this one moves: neither is touched
  for (int j = threadIdx.x; ok && j < t.n_blocks; j += blockDim.x) {
    const long long c = t.blk[4 * j + 3], n = t.blk[4 * j + 1];
    if (j != b && n > 0 && t.blk[4 * j + 2] == row && c < ctx + T && ctx < c + n) ok = false;
  }
  if (ok)
    for (int j = threadIdx.x; j <= acc; j += blockDim.x) {
      const int p = path[(size_t)b * t.max_nodes + j], before = j ? path[(size_t)b * t.max_nodes + j - 1] : -1;
      if (p <= before || p >= T) ok = false;
      src[j] = (int16_t)p;
      if (p != j) atomicMin(&first, j);   // the slots before the first gap stay where they are
    }
  ok = __syncthreads_and(ok);
  if (!ok) {
    if (threadIdx.x == 0) set_status(status, kStatusBadIndex);
    return;
  }
  const int j0 = max(first, 1);
  if (j0 > acc) return;
  const int cols = slot_bytes / 16;
  const long long n_vec = (long long)n_layers * n_kv_heads * cols * 2;
  const long long n_exp = ke ? (long long)n_layers * n_kv_heads * 2 : 0;
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n_vec) {
    const int col = (int)(i % cols), h = (int)(i / cols % n_kv_heads);
    const long long lk = i / cols / n_kv_heads;
    uint8_t* base = (lk & 1 ? v : k);
    uint4* p = reinterpret_cast<uint4*>(base + ((((size_t)(lk >> 1) * max_batch + row) * n_kv_heads + h) * max_seq + ctx) * slot_bytes) + col;
    for (int j = j0; j <= acc; j += 4) {
      uint4 buf[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j + u <= acc) buf[u] = p[(size_t)src[j + u] * cols];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j + u <= acc) p[(size_t)(j + u) * cols] = buf[u];
    }
  } else if (i < n_vec + n_exp) {
    const long long e = i - n_vec;
    const int h = (int)(e % n_kv_heads);
    const long long lk = e / n_kv_heads;
    uint8_t* p = (lk & 1 ? ve : ke) + (((size_t)(lk >> 1) * max_batch + row) * n_kv_heads + h) * max_seq + ctx;
    for (int j = j0; j <= acc; ++j) p[j] = p[src[j]];
  }
}

template <typename T, int FMT>
cudaError_t append_d(int D, int n_tok, cudaStream_t s, const T* qkv, int ld, T* q_out, int ldo, int H, const int32_t* pos,
                     const int32_t* slot, const int32_t* row, const CacheGeom& g, const float* cs, const float* sn, int rl, int* st) {
  if (D == 64)
    return launch_pdl(kv_append_kernel<T, FMT, 64>, dim3(n_tok), dim3(256), 0, s, qkv, ld, q_out, ldo, H, pos, slot, row, g, cs, sn, rl, st);
  return launch_pdl(kv_append_kernel<T, FMT, 128>, dim3(n_tok), dim3(256), 0, s, qkv, ld, q_out, ldo, H, pos, slot, row, g, cs, sn, rl, st);
}
template <typename T>
cudaError_t append_t(int fmt, int D, int n_tok, cudaStream_t s, void* qkv, int ld, void* q_out, int ldo, int H, const int32_t* pos,
                     const int32_t* slot, const int32_t* row, const CacheGeom& g, const float* cs, const float* sn, int rl, int* st) {
  const T* x = static_cast<const T*>(qkv);
  T* q = static_cast<T*>(q_out);
  if (fmt == EESD_KV_E4M3) return append_d<T, EESD_KV_E4M3>(D, n_tok, s, x, ld, q, ldo, H, pos, slot, row, g, cs, sn, rl, st);
  if (fmt == EESD_KV_INT8) return append_d<T, EESD_KV_INT8>(D, n_tok, s, x, ld, q, ldo, H, pos, slot, row, g, cs, sn, rl, st);
  return append_d<T, EESD_KV_MODEL>(D, n_tok, s, x, ld, q, ldo, H, pos, slot, row, g, cs, sn, rl, st);
}

template <typename T, int FMT>
cudaError_t read_d(int D, dim3 grid, cudaStream_t s, const CacheGeom& g, const int32_t* slot, const int32_t* row, int n, void* k,
                   void* v, int* st) {
  if (D == 64)
    return launch_pdl(kv_read_kernel<T, FMT, 64>, grid, dim3(256), 0, s, g, slot, row, n, static_cast<T*>(k), static_cast<T*>(v), st);
  return launch_pdl(kv_read_kernel<T, FMT, 128>, grid, dim3(256), 0, s, g, slot, row, n, static_cast<T*>(k), static_cast<T*>(v), st);
}
template <typename T>
cudaError_t read_t(int fmt, int D, dim3 grid, cudaStream_t s, const CacheGeom& g, const int32_t* slot, const int32_t* row, int n,
                   void* k, void* v, int* st) {
  if (fmt == EESD_KV_E4M3) return read_d<T, EESD_KV_E4M3>(D, grid, s, g, slot, row, n, k, v, st);
  if (fmt == EESD_KV_INT8) return read_d<T, EESD_KV_INT8>(D, grid, s, g, slot, row, n, k, v, st);
  return read_d<T, EESD_KV_MODEL>(D, grid, s, g, slot, row, n, k, v, st);
}

int launched(const char* who, cudaError_t e) {
  return e == cudaSuccess ? EESD_OK : fail_arg(EESD_ERR_CUDA, "%s: launch: %s", who, cudaGetErrorString(e));
}

}  // namespace
}  // namespace eesd

using namespace eesd;

extern "C" {

int eesd_tree_meta(const EesdTree* t, int max_batch, int max_seq, int32_t* status, void* stream) {
  int rc = check_tree("tree_meta", t);
  if (rc) return rc;
  if (max_batch <= 0 || max_seq <= 0) return fail_arg(EESD_ERR_ARG, "tree_meta: cache sizes");
  if (t->n_tokens == 0 || t->n_blocks == 0) return EESD_OK;
  if (!t->tok_pos || !t->tok_slot || !t->tok_row) return fail_arg(EESD_ERR_ARG, "tree_meta: null output");
  if (t->parent && t->max_nodes > EESD_TREE_MAX_NODES)
    return fail_arg(EESD_ERR_ARG, "tree_meta: parents need max_nodes <= %d", EESD_TREE_MAX_NODES);
  if ((rc = check_stream("tree_meta", stream))) return rc;
  return launched("tree_meta", launch_pdl(tree_meta_kernel, dim3(t->n_blocks), dim3(128), 0, static_cast<cudaStream_t>(stream), *t,
                                          max_batch, max_seq, status));
}

int eesd_kv_append(int dtype, const EesdKvCache* c, int layer, void* qkv, int ld_qkv, int n_heads, const int32_t* tok_pos,
                   const int32_t* tok_slot, const int32_t* tok_row, int n_tok, const float* rope_cos, const float* rope_sin,
                   int rope_len, void* q_out, int32_t* status, void* stream) {
  int rc = check_cache("kv_append", dtype, c, layer);
  if (rc) return rc;
  if (n_tok < 0 || rope_len <= 0 || n_heads <= 0 || n_heads % c->n_kv_heads)
    return fail_arg(EESD_ERR_ARG, "kv_append: n_tok %d, rope_len %d, heads %d / %d", n_tok, rope_len, n_heads, c->n_kv_heads);
  if (n_tok == 0) return EESD_OK;
  if (!qkv || !tok_pos || !tok_row || !rope_cos || !rope_sin) return fail_arg(EESD_ERR_ARG, "kv_append: null argument");
  if (ld_qkv % 8 || ld_qkv < (n_heads + 2 * c->n_kv_heads) * c->head_dim)
    return fail_arg(EESD_ERR_ARG, "kv_append: ld_qkv %d (a multiple of 8, at least the fused row)", ld_qkv);
  if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(rope_cos) |
       reinterpret_cast<uintptr_t>(rope_sin)) & 15)
    return fail_arg(EESD_ERR_ARG, "kv_append: qkv, q_out and the RoPE tables must be 16-byte aligned");
  if ((rc = check_stream("kv_append", stream))) return rc;
  const CacheGeom g = cache_layer(c, dtype, layer);
  const int ldo = q_out ? n_heads * c->head_dim : ld_qkv;
  void* qo = q_out ? q_out : qkv;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int32_t* slot = tok_slot ? tok_slot : tok_pos;
  const cudaError_t e =
      dtype == EESD_BF16
          ? append_t<bf16>(c->format, c->head_dim, n_tok, s, qkv, ld_qkv, qo, ldo, n_heads, tok_pos, slot, tok_row, g, rope_cos, rope_sin, rope_len, status)
          : append_t<float>(c->format, c->head_dim, n_tok, s, qkv, ld_qkv, qo, ldo, n_heads, tok_pos, slot, tok_row, g, rope_cos, rope_sin, rope_len, status);
  return launched("kv_append", e);
}

int eesd_kv_read(int dtype, const EesdKvCache* c, int layer, const int32_t* tok_slot, const int32_t* tok_row, int n_tok, void* k_out,
                 void* v_out, int32_t* status, void* stream) {
  int rc = check_cache("kv_read", dtype, c, layer);
  if (rc) return rc;
  if (n_tok < 0) return fail_arg(EESD_ERR_ARG, "kv_read: n_tok %d", n_tok);
  if (n_tok == 0 || (!k_out && !v_out)) return EESD_OK;
  if (!tok_slot || !tok_row) return fail_arg(EESD_ERR_ARG, "kv_read: null argument");
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15)
    return fail_arg(EESD_ERR_ARG, "kv_read: outputs must be 16-byte aligned");
  if ((rc = check_stream("kv_read", stream))) return rc;
  const CacheGeom g = cache_layer(c, dtype, layer);
  const int ctas = n_tok / 8 + (n_tok % 8 != 0);                         // 8 warps each, a token per warp
  const dim3 grid((unsigned)(ctas < 148 * 16 ? ctas : 148 * 16), (k_out && v_out) ? 2 : 1);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == EESD_BF16 ? read_t<bf16>(c->format, c->head_dim, grid, s, g, tok_slot, tok_row, n_tok, k_out, v_out, status)
                                           : read_t<float>(c->format, c->head_dim, grid, s, g, tok_slot, tok_row, n_tok, k_out, v_out, status);
  return launched("kv_read", e);
}

int eesd_tree_accept(const int32_t* y, const int32_t* ids, const EesdTree* t, int32_t* path, int32_t* n_acc, int32_t* next,
                     int32_t* status, void* stream) {
  int rc = check_tree("tree_accept", t);
  if (rc) return rc;
  if (t->n_tokens == 0 || t->n_blocks == 0) return EESD_OK;
  if (!y || !ids || !path || !n_acc || !next) return fail_arg(EESD_ERR_ARG, "tree_accept: null argument");
  if (t->max_nodes > EESD_TREE_MAX_NODES)
    return fail_arg(EESD_ERR_ARG, "tree_accept: max_nodes %d (at most %d)", t->max_nodes, EESD_TREE_MAX_NODES);
  if ((rc = check_stream("tree_accept", stream))) return rc;
  return launched("tree_accept", launch_pdl(tree_accept_kernel, dim3(t->n_blocks), dim3(32), 0, static_cast<cudaStream_t>(stream), *t,
                                            y, ids, path, n_acc, next, status));
}

int eesd_kv_compact(int dtype, const EesdKvCache* c, const EesdTree* t, const int32_t* path, const int32_t* n_acc, int32_t* status,
                    void* stream) {
  int rc = check_cache("kv_compact", dtype, c, 0);
  if (!rc) rc = check_tree("kv_compact", t);
  if (rc) return rc;
  if (t->n_tokens == 0 || t->n_blocks == 0) return EESD_OK;
  if (!path || !n_acc) return fail_arg(EESD_ERR_ARG, "kv_compact: null argument");
  if (t->max_nodes > EESD_TREE_MAX_NODES)
    return fail_arg(EESD_ERR_ARG, "kv_compact: max_nodes %d (at most %d)", t->max_nodes, EESD_TREE_MAX_NODES);
  if ((rc = check_stream("kv_compact", stream))) return rc;
  const int slot_bytes = c->head_dim * (int)cache_elem_bytes(c, dtype);
  const bool q8 = c->format != EESD_KV_MODEL;
  const long long n = (long long)c->n_layers * c->n_kv_heads * 2 * (slot_bytes / 16 + (q8 ? 1 : 0));
  return launched("kv_compact",
                  launch_pdl(kv_compact_kernel, dim3((unsigned)((n + 255) / 256), t->n_blocks), dim3(256), 0,
                             static_cast<cudaStream_t>(stream), static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v),
                             q8 ? c->k_exp : nullptr, q8 ? c->v_exp : nullptr, c->n_layers, c->n_kv_heads, c->max_batch, c->max_seq,
                             slot_bytes, *t, path, n_acc, status));
}

}  // extern "C"
