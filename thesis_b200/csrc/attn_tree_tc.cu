// Tree attention for many query rows per KV head (wide trees, prefill chunks): tcgen05.
//
// A persistent CTA per SM works on row tiles of up to 256 rows (two M = 128 accumulators).  All (block, row tile,
// KV head) units are laid end to end in 64-key tiles and cut into equal runs, one per CTA, so ragged contexts and
// causal tiles balance whatever their number; a unit that a cut goes through leaves normalised partial outputs,
// which a second kernel joins in order.
//
// Per 64-key tile: S = Q K^T, softmax weights P from S in registers into TMEM, O += P V, K and V in shared memory in the
// layout they arrive in (V is the MN-major operand).  Operands in TMEM issue faster than from shared memory (42
// against 75 clocks for N = 64), so P and the first 128 rows of Q are there; the other 128 rows of Q have no room
// left beside two fp32 O (256 columns) and two S and P (192).  Two streams alternate, and S of a stream's next tile is
// computed while its softmax still works on this one: with more than 128 rows each stream is one half of the rows
// over all key tiles; with fewer, both share the rows and take every other key tile, and meet at the end.
//
// 8-bit caches: a warpgroup turns the TMA-loaded bytes into the f16 tiles that the products read, each key's power of
// two relative to the tile's largest multiplied in (exact: K's within 2^16, V's within 2^8 of each other), so the softmax sees
// one scale per tile.  Scales that lie further apart stay out of the operands and multiply scores and weights instead, and so
// do V's in tiles that some row does not wholly see: what a row does not see must not decide its precision.
//
// Roles of the 20 warps: 0 TMA, 1 and 3 MMA issue of stream 0 and 1 (a satisfied barrier wait costs some 150 clocks,
// and each tile takes four of them), 2 the schedule, 4-7 and 8-11 softmax of stream 0 and 1 (a thread is a row),
// 12-15 and 16-19 conversion of K and of V (8-bit), or 12-15 the check of V tiles that some row does not wholly see (bf16).
//
// Measured (32 query and 8 KV heads of 128): 48 nodes at 131 k slots over int8 192 us, 536 TFLOP/s, 1.41 TB/s; four 512-token
// chunks at up to 3.6 k slots over e4m3 136 us, 507 TFLOP/s, over bf16 110 us, 624 TFLOP/s; 16 trees of 31 nodes at 1 k to 4 k slots
// over e4m3 66 us, over bf16 53 us.  By the clock, in a copy that recorded it, a pair
// of 128-row tiles takes some 2800 clocks per 64 keys, of which the products are 1000 and the exponentials 1024: what
// bounds it is the chain wait, load, maximum, exponentials, store of the one softmax warp that a stream has per scheduler.
// One row tile is bound by the conversion (1900 clocks a tile) and by the units' starts and ends, 7 k clocks each.  Tried and
// slower: two warpgroups each for the conversion of K and V (tree 64 -> 70 us, long 190 -> 206: fewer registers).
#include <algorithm>

#include "attn_tree.h"
#include "attn_tree_dev.cuh"
#include "attn_tree_tc.h"
#include "gemm_tc.h"
#include "kernels.h"

namespace eesd {
namespace {

constexpr int KT = 64;                     // keys per tile
constexpr int kThreads = 640;
constexpr uint32_t kColO = 0, kColQ = 256;                // TMEM columns; O of stream x at 128 x
constexpr uint32_t kColS = 320, kColP = 384, kSP = 96;    // S and P of stream x add kSP x

// One arrival per warp, after all of its lanes: an arrival is an atomic on shared memory, and 32 of them on one
// barrier serialise.
__device__ __forceinline__ void mbar_arrive(uint32_t bar);
__device__ __forceinline__ void warp_arrive(void* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(bar));
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void bulk_prefetch_l2(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}
// One lane of a converged warp.  The branch on it keeps the warp's scalar registers usable, which a branch on the
// lane number does not: a product then issues every 42 clocks (N = 64) instead of every 118.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.b32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p != 0;
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
#define EESD_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define EESD_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 32 lanes x 32 columns; lane i of the warp holds TMEM lane (quadrant base + i)
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : EESD_R8(r, 0), EESD_R8(r, 8), EESD_R8(r, 16), EESD_R8(r, 24)
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : EESD_R8(r, 0), EESD_R8(r, 8)
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::EESD_W8(r, 0), EESD_W8(r, 8),
      "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
      "%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::EESD_W8(r, 0),
      EESD_W8(r, 8), EESD_W8(r, 16), EESD_W8(r, 24), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Whether the phase is complete, now (try_wait may stay for a while)
__device__ __forceinline__ bool mbar_test_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred P;\n\tmbarrier.test_wait.parity.shared::cta.b64 P, [%1], %2;\n\tselp.b32 %0, 1, 0, P;\n\t}"
               : "=r"(ok)
               : "r"(bar), "r"(parity)
               : "memory");
  return ok != 0;
}
// The whole warp waits and goes on together (what follows are warp-wide instructions).
__device__ __forceinline__ bool warp_wait(const void* bar, uint32_t parity, volatile int* abort_flag, uint32_t limit) {
  if (__builtin_expect(__all_sync(0xffffffffu, mbar_try_wait(smem_u32(bar), parity)), 1)) return true;
  return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, abort_flag, limit));
}
template <int N> __device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// two fp32 operations at once
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack_f2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack_f2(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// MN-major operand tile (64-element, 128-byte rows of the MN index per K index, 128-byte swizzle): 8 K indices
// are 1024 bytes (stride), the next 64 MN elements lie `lbo` bytes on.
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t smem_addr, uint32_t lbo) {
  return sw128_kmajor_desc(smem_addr) & ~((uint64_t)0x3FFF << 16) | (uint64_t)((lbo >> 4) & 0x3FFF) << 16;
}
// M = 128 x N, fp32 accumulate; f16 or bf16 operands, B K-major or MN-major
template <int FMT> __device__ __forceinline__ uint32_t idesc_f32(int n, bool b_mn) {
  const uint32_t ab = FMT == EESD_KV_MODEL ? (1u << 7 | 1u << 10) : 0u;
  return (1u << 4) | ab | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

// ------------------------------------------------------------------ the flat schedule
// Entry e = (block, row tile); its unit of each KV head takes `tiles` key tiles.  On the flat axis a unit is kUnitCost
// positions (what starting a unit costs, in tiles) and then its tiles; entries follow one another, their heads inside.
// Measured with 4, 6, 8, 10 (us): four 512-token chunks over e4m3 174, 141, 136, 137, over bf16 114, 112, 110, 112; 16 trees of 31
// nodes over e4m3 68.8, 66.6, 65.8, 67.1, over bf16 53.8, 52.7, 52.5, 52.7; nine 235-token chunks over int8 78, 76, 75, 73; 48 nodes at
// 131 k slots and 16 trees of 48 at 400 the same with all.
constexpr int kUnitCost = 8;
struct Entry {
  BlockInfo bi;
  int r0, nrows, n_keys, all_see, tiles;   // slots below all_see are seen by every row of the tile
  __device__ int length() const { return tiles ? tiles + kUnitCost : 0; }
};
__device__ __forceinline__ Entry entry_of(const TreeGeom& g, const CacheGeom& c, const TcSchedule& sc, int e, bool& bad) {
  Entry x;
  const int b = e / sc.tiles_max, tile = e - b * sc.tiles_max;
  x.tiles = 0;
  bad = !block_fits(g, c, b, x.bi);
  if (bad) return x;
  x.r0 = tile * sc.rows;
  x.nrows = min(sc.rows, x.bi.T * g.G - x.r0);
  if (x.nrows <= 0) return x;
  x.n_keys = x.bi.ctx + (g.mask ? x.bi.T : (x.r0 + x.nrows - 1) / g.G + 1);
  x.all_see = x.bi.ctx + (g.mask ? 0 : x.r0 / g.G + 1);
  x.tiles = (x.n_keys + KT - 1) / KT;
  return x;
}
struct Piece : Entry {
  int h, t0, t1, index;     // KV head, key tiles [t0, t1), number of the piece in its CTA
  long long u0;             // flat position of the unit
  __device__ bool whole() const { return t0 == 0 && t1 == tiles; }
};
// The pieces of one CTA's run [pos, end).  With a fixed split (sc.chunk_tiles) a unit is cut at multiples of it and
// a piece belongs to the CTA whose run holds its first position; otherwise a piece is what the run holds of a unit.
struct PieceIter {
  long long pos, end, base;
  int e, index, loaded;
  __device__ bool next(const TreeGeom& g, const CacheGeom& c, const TcSchedule& sc, Piece& p) {
#pragma unroll 1
    while (pos < end) {
      if (loaded != e) {
        bool bad;
        static_cast<Entry&>(p) = entry_of(g, c, sc, e, bad);
        loaded = e;
      }
      const int len = p.length();
      const long long span = (long long)len * c.n_kv_heads;
      if (pos >= base + span) {
        base += span;
        ++e;
        continue;
      }
      const int in = (int)(pos - base);
      p.h = in / len;
      p.u0 = base + (long long)p.h * len;
      const int off = (int)(pos - p.u0);
      if (sc.chunk_tiles) {
        p.t0 = off == 0 ? 0 : (max(off - kUnitCost, 1) + sc.chunk_tiles - 1) / sc.chunk_tiles * sc.chunk_tiles;
        p.t1 = min(p.tiles, p.t0 + sc.chunk_tiles);
        if (p.t0 < p.tiles && p.u0 + (p.t0 ? kUnitCost + p.t0 : 0) >= end) return false;
      } else {
        p.t0 = max(off - kUnitCost, 0);
        p.t1 = (int)max(0LL, min((long long)p.tiles, end - p.u0 - kUnitCost));
      }
      pos = p.u0 + kUnitCost + min(p.t1, p.tiles);
      if (p.t0 >= p.t1) {                                  // a run that ends before the unit's first tile
        if (!sc.chunk_tiles) return false;
        pos = p.u0 + len;
        continue;
      }
      p.index = index++;
      return true;
    }
    return false;
  }
};

// Four stored bytes as f16 pairs times the half pair m: exact unpacking, then one product (e4m3) or, with the offset of
// the integer trick folded in, one FMA: (1024 + u) m - 1152 m, u = element + 128 (int8; m at most 2^5 keeps 1152 m finite).
template <int FMT> struct Scaler {
  __half2 m, off;
  __device__ explicit Scaler(uint32_t bits) {
    m = *reinterpret_cast<const __half2*>(&bits);
    off = FMT == EESD_KV_INT8 ? __hmul2(m, __halves2half2(__ushort_as_half(0xe480), __ushort_as_half(0xe480))) : m;   // -1152 m
  }
  __device__ void operator()(uint32_t w, uint32_t& lo, uint32_t& hi) const {
    if constexpr (FMT == EESD_KV_INT8) {
      w ^= 0x80808080u;
      const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
      const __half2 x = __hfma2(*reinterpret_cast<const __half2*>(&a), m, off), y = __hfma2(*reinterpret_cast<const __half2*>(&b), m, off);
      lo = *reinterpret_cast<const uint32_t*>(&x);
      hi = *reinterpret_cast<const uint32_t*>(&y);
    } else {
      unpack4<FMT>(w, lo, hi);
      const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&lo), m), y = __hmul2(*reinterpret_cast<const __half2*>(&hi), m);
      lo = *reinterpret_cast<const uint32_t*>(&x);
      hi = *reinterpret_cast<const uint32_t*>(&y);
    }
  }
};

template <int FMT> constexpr int kUp = FMT == EESD_KV_E4M3 ? 14 : 5;   // a tile's largest 8-bit elements in f16: 28672, 4064
template <int D, int FMT> struct TcShape {
  static constexpr bool Q8 = FMT != EESD_KV_MODEL;
  static constexpr int TILE = KT * D * 2;              // bytes of one 16-bit K (or V) tile
  static constexpr int RAW = KT * D * 2;               // 8-bit: K and V bytes of one tile
  // 16-bit K / V stages.  Even: with one row tile each stream waits for every other tile only, and a stage that both used in turn
  // would have it wait for a phase whose predecessor, the other stream's tile, may not have landed: a parity wait then returns at once.
  static constexpr int NS = Q8 ? 2 : 4;
  static_assert(NS % 2 == 0, "a stage belongs to one stream");
  static constexpr int RS = Q8 ? 6 : 0;                // raw stages
  static constexpr int FR = 8;                         // factor ring: six tiles can be between conversion and softmax
  static constexpr int QB = 128 * D * 2 + 128 * 128;   // Q of stream 1 (more than 128 rows), half rows on their way to TMEM
  static constexpr size_t ctl = 16384;
  static constexpr size_t smem = 1024 + (size_t)2 * NS * TILE + (size_t)RS * RAW + QB + ctl;
};
constexpr int kPieces = 4;                 // pieces between the schedule warp and the slowest role
constexpr int kReaders = 19;               // warps that read them: TMA, 2 MMA, 8 softmax, 8 conversion
enum : int { kHowK = 1 << 8, kHowV = 1 << 9 };
struct TcControl {
  uint64_t kfull[4], kempty[4], vfull[4], vempty[4], vclean[4], raw_full[6], raw_empty[6];
  uint64_t piece_full[kPieces], piece_empty[kPieces];
  Piece piece[kPieces];                    // tiles == 0: there are no more
  uint64_t s_full[2], s_free[2], p_ready[2], pv_done[2], q_ready, o_done, ml_ready, epi_done, drain[2];
  // 8-bit, per tile: ref is V's largest exponent byte, kt the one factor of its keys, and how (kHow*, above ref's byte) what is not in
  // the operands.  Keyed K: 2^ek of the keys multiplies the scores.  Keyed V: 2^ev of the keys multiplies the weights, ev is the exponent
  // byte (0 for NaN and slots past the end).
  alignas(16) float fk[8][KT];
  alignas(16) float fv[8][KT];
  float kt[8];
  alignas(16) uint8_t ev[8][KT];
  alignas(16) uint8_t exps[6][2 * KT];     // raw exponent bytes, K then V
  int ref[8];
  uint32_t nan[8][2];                      // keys whose V is NaN
  float ml[2][2][3][128];                  // one row tile: max, sum and eref of the streams (by piece parity)
  long long lo, hi, base, run;
  long long wsum[20];
  uint32_t tmem;
  int e0;
  int abort, dropped;
};
static_assert(sizeof(TcControl) <= 16384 && alignof(TcControl) <= 16, "control block");

template <int D, int FMT>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tree_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, TreeGeom g, CacheGeom c,
                        TcSchedule sc, const bf16* __restrict__ q, bf16* __restrict__ out) {
  using S = TcShape<D, FMT>;
  constexpr bool Q8 = S::Q8;
  constexpr int NS = S::NS, RS = Q8 ? S::RS : 1, FR = S::FR, HALVES = D / 64;
  pdl_trigger();
  pdl_wait();
  extern __shared__ uint8_t smem8[];
  uint8_t* sm = smem8 + (-smem_u32(smem8) & 1023);     // an offset, so that the compiler still knows it as shared memory
  const uint32_t kbuf = smem_u32(sm), vbuf = kbuf + NS * S::TILE, raw = vbuf + NS * S::TILE, qbuf = raw + S::RS * S::RAW,
                 qstage = qbuf + 128 * D * 2;
  TcControl& ct = *reinterpret_cast<TcControl*>(sm + 2 * NS * S::TILE + S::RS * S::RAW + S::QB);
  volatile int* abort_flag = &ct.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // ---- this CTA's run of the flat schedule: block-wide prefix of the entries' tiles
  {
    const int E = sc.entries, seg = (E + kThreads - 1) / kThreads;
    const int a = min(E, tid * seg), b = min(E, a + seg);
    long long sum = 0;
#pragma unroll 1
    for (int e = a; e < b; ++e) {
      bool bad;
      sum += entry_of(g, c, sc, e, bad).length();
      if (bad && blockIdx.x == 0) set_status(g.status, kStatusBadIndex);
    }
    long long inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) ct.wsum[warp] = inc;
    if (tid == 0) {
      ct.abort = ct.dropped = 0;
      ct.e0 = E;
      for (int i = 0; i < NS; ++i) {
        mbar_init(smem_u32(&ct.kfull[i]), Q8 ? 4 : 1);
        mbar_init(smem_u32(&ct.vfull[i]), Q8 ? 4 : 1);
        mbar_init(smem_u32(&ct.kempty[i]), 2);
        mbar_init(smem_u32(&ct.vempty[i]), 2);
        mbar_init(smem_u32(&ct.vclean[i]), 4);
      }
      for (int i = 0; i < RS; ++i) {
        mbar_init(smem_u32(&ct.raw_full[i]), 1);
        mbar_init(smem_u32(&ct.raw_empty[i]), 8);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(smem_u32(&ct.s_full[i]), 1);
        mbar_init(smem_u32(&ct.s_free[i]), 4);
        mbar_init(smem_u32(&ct.p_ready[i]), 4);
        mbar_init(smem_u32(&ct.pv_done[i]), 1);
      }
      for (int i = 0; i < kPieces; ++i) {
        mbar_init(smem_u32(&ct.piece_full[i]), 1);
        mbar_init(smem_u32(&ct.piece_empty[i]), kReaders);
      }
      mbar_init(smem_u32(&ct.q_ready), 8);
      mbar_init(smem_u32(&ct.ml_ready), 9);                            // the softmax warps, and stream 1's issuing thread
      mbar_init(smem_u32(&ct.epi_done), 8);
      mbar_init(smem_u32(&ct.o_done), 2);
      mbar_init(smem_u32(&ct.drain[0]), 1);
      mbar_init(smem_u32(&ct.drain[1]), 1);
      fence_mbar_init();
    }
    if (warp == 1) {
      tmem_alloc(smem_u32(&ct.tmem), 512);
      tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    long long before = inc - sum, total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      const long long v = ct.wsum[w];
      if (w < warp) before += v;
      total += v;
    }
    const int Hkv = c.n_kv_heads;
    const long long W = total * Hkv, n = gridDim.x;
    const long long run = max(1LL, W < (1LL << 31) - n ? (long long)((uint32_t)(W + n - 1) / (uint32_t)n) : (W + n - 1) / n), lo = min(W, blockIdx.x * run), hi = min(W, lo + run);
    if (tid == 0) {
      ct.lo = lo;
      ct.hi = hi;
      ct.run = run;
      sc.cuts[blockIdx.x].nrows = 0;                                    // no unit of this run goes on in the next one
    }
    if (lo >= before * Hkv && lo < (before + sum) * Hkv) {
      long long base = before * Hkv;
#pragma unroll 1
      for (int e = a; e < b; ++e) {
        bool bad;
        const long long span = (long long)entry_of(g, c, sc, e, bad).length() * Hkv;
        if (lo >= base && lo < base + span) {
          ct.e0 = e;
          ct.base = base;
        }
        base += span;
      }
    }
    __syncthreads();
  }
  // Every role reads its pieces, in order, from the ring that warp 2 fills.
  auto piece_wait = [&](int k) { return mbar_wait(smem_u32(&ct.piece_full[k % kPieces]), k / kPieces & 1, abort_flag, g.spin); };
  auto piece_free = [&](int k) { mbar_arrive(smem_u32(&ct.piece_empty[k % kPieces])); };
  const uint32_t tmem = ct.tmem;

  if (warp < 4) reg_dec<56>();
  if (warp == 0) {
    // ------------------------------------------------------------ TMA
    if (elect_one()) {
      int cnt = 0, k_issued = 0, v_issued = 0;
      bool ok = true;
      tma_prefetch_desc(&kmap);
      tma_prefetch_desc(&vmap);
#pragma unroll 1
      for (int k = 0; (ok = piece_wait(k)); ++k) {
        const Piece& p = ct.piece[k % kPieces];
        if (p.tiles == 0) break;
        const int slot0 = (int)cache_slot(c, p.bi.row, p.h, 0);
#pragma unroll 1
        for (int t = p.t0; t < p.t1; ++t, ++cnt) {
          if constexpr (Q8) {
            const int s = cnt % RS;
            if (!(ok = mbar_wait(smem_u32(&ct.raw_empty[s]), (cnt / RS & 1) ^ 1, abort_flag, g.spin))) break;
            const uint32_t fb = smem_u32(&ct.raw_full[s]), dst = raw + s * S::RAW, ex = smem_u32(ct.exps[s]);
            const uint32_t eb = min(KT, c.max_seq - t * KT);          // max_seq % 16 == 0
            mbar_arrive_expect_tx(fb, S::RAW + 2 * eb);
            tma_load_2d(dst, &kmap, 0, slot0 + t * KT, fb);
            tma_load_2d(dst + S::RAW / 2, &vmap, 0, slot0 + t * KT, fb);
            bulk_g2s(ex, c.ke + slot0 + t * KT, eb, fb);
            bulk_g2s(ex + KT, c.ve + slot0 + t * KT, eb, fb);
            k_issued = cnt + 1;
          } else {
            const int s = cnt % NS;
            const uint32_t ph = (cnt / NS & 1) ^ 1;
            if (!(ok = mbar_wait(smem_u32(&ct.kempty[s]), ph, abort_flag, g.spin))) break;
            const uint32_t kb = smem_u32(&ct.kfull[s]), vb = smem_u32(&ct.vfull[s]);
            mbar_arrive_expect_tx(kb, S::TILE);
            for (int h = 0; h < HALVES; ++h) tma_load_2d(kbuf + s * S::TILE + h * KT * 128, &kmap, h * 64, slot0 + t * KT, kb);
            k_issued = cnt + 1;
            if (!(ok = mbar_wait(smem_u32(&ct.vempty[s]), ph, abort_flag, g.spin))) break;
            mbar_arrive_expect_tx(vb, S::TILE);
            for (int h = 0; h < HALVES; ++h) tma_load_2d(vbuf + s * S::TILE + h * KT * 128, &vmap, h * 64, slot0 + t * KT, vb);
            v_issued = cnt + 1;
          }
        }
        if (!ok) break;
        piece_free(k);
      }
      if (!ok) {
        set_status(g.status, kStatusTimeoutProducer);
        *abort_flag = 1;
      }
      // Nothing may be in flight when the CTA exits, and after an abort, perhaps one that is still to come, nobody else waits
      // for what has been issued: the last load of every stage is waited for here.
      for (int i = max(0, k_issued - (Q8 ? RS : NS)); i < k_issued; ++i)
        mbar_drain(Q8 ? smem_u32(&ct.raw_full[i % RS]) : smem_u32(&ct.kfull[i % NS]), (i / (Q8 ? RS : NS)) & 1);
      for (int i = max(0, v_issued - NS); i < v_issued; ++i) mbar_drain(smem_u32(&ct.vfull[i % NS]), (i / NS) & 1);
    }
  } else if (warp == 1 || warp == 3) {
    // ------------------------------------------------------------ MMA issue of stream x
    if (elect_one()) {
      const int x = warp >> 1;
      const uint32_t id_qk = idesc_f32<FMT>(KT, false), id_pv = idesc_f32<FMT>(D, true);
      const uint32_t dS = tmem + kColS + x * kSP, dO = tmem + kColO + x * 128, aP = tmem + kColP + x * kSP;
      int cnt0 = 0, piece = 0, n_q = 0, n_p = 0;
      bool ok = true, issued = false;
#pragma unroll 1
      for (; (ok = piece_wait(piece)); ++piece) {
        const Piece& p = ct.piece[piece % kPieces];
        if (p.tiles == 0) break;
        const int nt = p.t1 - p.t0;
        const bool two = p.nrows > 128;
        const int step = two ? 1 : 2, t0 = two ? 0 : x;
        // with one row tile a key tile has this stream only: it frees the stage for both
        auto free_stage = [&](uint64_t* bar) {
          tc_commit(smem_u32(bar));
          if (!two) tc_commit(smem_u32(bar));
        };
        if (!(ok = mbar_wait(smem_u32(&ct.q_ready), piece & 1, abort_flag, g.spin))) break;
        // With one key tile stream 1 has no product that the softmax would wait for: it says that it has seen this Q, or the next
        // one's phase could end before it looks, and it would wait for good.
        if (!two && x == 1) mbar_arrive(smem_u32(&ct.ml_ready));
        // S of the stream's next tile as soon as the last one is in registers, then O of the last one when its softmax ends
#pragma unroll 1
        for (int i = t0 - step; i < nt; i += step) {
          const int j = i + step;
          if (j < nt) {
            const int cnt = cnt0 + j, st = cnt % NS;
            if (n_q && !(ok = mbar_wait(smem_u32(&ct.s_free[x]), (n_q - 1) & 1, abort_flag, g.spin))) break;
            ++n_q;
            if (!(ok = mbar_wait(smem_u32(&ct.kfull[st]), cnt / NS & 1, abort_flag, g.spin))) break;
            tc_fence_after();
            issued = true;
            const uint64_t kd = sw128_kmajor_desc(kbuf + st * S::TILE);
            if (two && x == 1) {
              const uint64_t qd = sw128_kmajor_desc(qbuf);
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)
                tc_mma_f16(dS, qd + (kk >> 2) * (128 * 128 >> 4) + (kk & 3) * 2, kd + (kk >> 2) * (KT * 128 >> 4) + (kk & 3) * 2, id_qk, kk > 0);
            } else {
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)
                tc_mma_ts(dS, tmem + kColQ + kk * 8, kd + (kk >> 2) * (KT * 128 >> 4) + (kk & 3) * 2, id_qk, kk > 0);
            }
            tc_commit(smem_u32(&ct.s_full[x]));
            free_stage(&ct.kempty[st]);
          }
          if (i >= 0) {
            const int cnt = cnt0 + i, st = cnt % NS;
            // The weights of a piece's first tile come after the last piece's output, so every earlier V has landed then.  Without
            // that a wait for V may be about the other stream's tile that the stage held before, and return at once; later
            // tiles' stages were this stream's own, and their V is asked for first, while the softmax works.
            if (i == t0 && !(ok = mbar_wait(smem_u32(&ct.p_ready[x]), n_p & 1, abort_flag, g.spin))) break;
            if (!(ok = mbar_wait(smem_u32(Q8 ? &ct.vfull[st] : &ct.vclean[st]), cnt / NS & 1, abort_flag, g.spin))) break;
            if (i != t0 && !(ok = mbar_wait(smem_u32(&ct.p_ready[x]), n_p & 1, abort_flag, g.spin))) break;
            ++n_p;
            tc_fence_after();
            const uint64_t vd = sw128_mnmajor_desc(vbuf + st * S::TILE, KT * 128);
#pragma unroll
            for (int kk = 0; kk < KT / 16; ++kk) tc_mma_ts(dO, aP + kk * 8, vd + kk * (16 * 128 >> 4), id_pv, i != t0 || kk > 0);
            tc_commit(smem_u32(&ct.pv_done[x]));
            free_stage(&ct.vempty[st]);
          }
        }
        if (!ok) break;
        tc_commit(smem_u32(&ct.o_done));
        cnt0 += nt;
        piece_free(piece);
      }
      if (!ok) {
        set_status(g.status, kStatusTimeoutMma);
        *abort_flag = 1;
      }
      if (issued) {                                                     // no product may be in flight at the end
        tc_commit(smem_u32(&ct.drain[x]));
        mbar_drain(smem_u32(&ct.drain[x]), 0);
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ the schedule
    if (elect_one()) {
      PieceIter it{ct.lo, ct.hi, ct.base, ct.e0, 0, -1};
      if (ct.e0 >= sc.entries) it.pos = it.end;
      bool ok = true;
      Piece p;
#pragma unroll 1
      for (int k = 0;; ++k) {
        if (!(ok = mbar_wait(smem_u32(&ct.piece_empty[k % kPieces]), (k / kPieces & 1) ^ 1, abort_flag, g.spin))) break;
        const bool more = it.next(g, c, sc, p);
        if (!more) p.tiles = 0;
        ct.piece[k % kPieces] = p;
        mbar_arrive(smem_u32(&ct.piece_full[k % kPieces]));
        if (!more) break;
        // its rows of q on their way to L2: a token's heads of the group lie together
        for (int node = p.r0 / g.G; node <= (p.r0 + p.nrows - 1) / g.G; ++node)
          bulk_prefetch_l2(q + (size_t)(p.bi.start + node) * g.ld_q + (size_t)p.h * g.G * D, g.G * D * 2);
      }
      if (!ok) {
        set_status(g.status, kStatusTimeoutProducer);
        *abort_flag = 1;
      }
    }
  } else if (warp >= 12) {
    reg_dec<48>();
    // ------------------------------------------------------------ conversion, or the check of V tiles
    const int ti = tid & 127;
    const bool is_v = warp >= 16;
    // The raw tile's bytes as f16, row r times 2^(e_r - top) (none below 2^-24; byte 255, a NaN, comes out as one);
    // top = 0: all rows times 2^flat; zeros from row `left` on.  A thread has one 16-byte chunk of every 16th (D = 64: 32nd) row; the 8 lanes of a
    // phase are on 8 rows and one chunk, conflict-free in both swizzles.
    constexpr int kChunks = D / 16, kRowStep = 128 / kChunks;
    const uint32_t ch = (uint32_t)ti / 8 % kChunks, row0 = (uint32_t)ti / (8 * kChunks) * 8 + (ti & 7);
    const uint32_t from = row0 * D + ((D == 128 ? ch ^ (row0 & 7) : ch ^ (row0 >> 1 & 3)) << 4);
    const uint32_t to0 = (ch >> 2) * (KT * 128) + row0 * 128 + ((2 * ch & 7 ^ (row0 & 7)) << 4), to1 = to0 ^ 16;
    [[maybe_unused]] auto convert = [&](const uint8_t* src, uint8_t* dst, const uint8_t* e, int top, int flat, int left) {
      // the warp's 32 rows' factors, one per lane
      static_assert(KT / kRowStep * 8 <= 32, "a warp's rows");
      const int mine = row0 + lane / 8 % (KT / kRowStep) * kRowStep, er = e[mine], x = top ? er - top : flat;
      const uint32_t h = mine >= left ? 0u : top && er == 255 ? 0x7fffu : x >= -14 ? (uint32_t)(x + 15) << 10 : x >= -24 ? 1u << (x + 24) : 0u;
      uint4 raw4[KT / kRowStep];                                        // all loads before the first store
#pragma unroll
      for (int i = 0; i < KT / kRowStep; ++i) raw4[i] = *reinterpret_cast<const uint4*>(src + from + i * (kRowStep * D));
#pragma unroll
      for (int i = 0; i < KT / kRowStep; ++i) {
        const uint4 w = raw4[i];
        const uint32_t m = __byte_perm(__shfl_sync(0xffffffffu, h, lane % 8 + 8 * i), 0, 0x1010);
        const Scaler<FMT> sc8(m);
        uint4 a, b;
        sc8(w.x, a.x, a.y);
        sc8(w.y, a.z, a.w);
        sc8(w.z, b.x, b.y);
        sc8(w.w, b.z, b.w);
        *reinterpret_cast<uint4*>(dst + to0 + i * (kRowStep * 128)) = a;
        *reinterpret_cast<uint4*>(dst + to1 + i * (kRowStep * 128)) = b;
      }
      fence_proxy_async_smem();
    };
    int cnt = 0;
    bool ok = true;
#pragma unroll 1
    for (int k = 0; (ok = __all_sync(0xffffffffu, piece_wait(k))); ++k) {
      const Piece& p = ct.piece[k % kPieces];
      if (p.tiles == 0) break;
#pragma unroll 1
      for (int t = p.t0; (Q8 || !is_v) && t < p.t1; ++t, ++cnt) {
        const int st = cnt % NS;
        if constexpr (Q8) {
          const int rs = cnt % RS, f = cnt % FR;
          if (!(ok = warp_wait(&ct.raw_full[rs], cnt / RS & 1, abort_flag, g.spin))) break;
          const bool partial = (t + 1) * KT > min(p.all_see, p.n_keys);
          const int left = p.n_keys - t * KT;
          // the largest exponents (of slots before the tile's end, NaN apart)
          const bool in0 = 2 * lane < left, in1 = 2 * lane + 1 < left;
          auto largest = [&](const uint8_t* e, int& a0, int& a1) {
            const uint32_t v = *reinterpret_cast<const uint16_t*>(e + 2 * lane);
            a0 = v & 255, a1 = v >> 8;
            return __reduce_max_sync(0xffffffffu, max(in0 && a0 != 255 ? a0 : 0, in1 && a1 != 255 ? a1 : 0));
          };
          // whether some scale lies more than 2^d below the largest (vectors at the smallest scale, zeros most often, apart)
          auto spread = [&](int em, int d, int a0, int a1) {
            return __any_sync(0xffffffffu, (in0 && a0 > 27 && a0 < em - d) || (in1 && a1 > 27 && a1 < em - d));
          };
          int a0, a1;
          const uint8_t *ek = ct.exps[rs], *ev = ek + KT;
          const int em = largest(is_v ? ev : ek, a0, a1);
          // Scales far apart stay out of the operand: K's where f16 would round (beyond 2^16), V's where what is small beside the
          // largest could matter all the same (beyond 2^8).  So do V's in a tile that some row does not wholly see: a slot that a row
          // does not see must not decide its precision.
          const bool keyed = spread(em, is_v ? 8 : 16, a0, a1) || (is_v && partial);
          const int top = keyed ? 0 : max(em, 27) - kUp<FMT>;
          int ref = 0;
          if (!is_v && warp == 12) {
            ref = largest(ev, a0, a1);
            ref |= (keyed ? kHowK : 0) | (spread(ref, 8, a0, a1) || partial ? kHowV : 0);
          }
          if (!(ok = warp_wait(is_v ? &ct.vempty[st] : &ct.kempty[st], (cnt / NS & 1) ^ 1, abort_flag, g.spin))) break;
          if (!is_v && warp == 12) {
            // What the softmax needs to know of the tile: it is there once S is.  The ring's last reader is behind the
            // products that freed this stage.
            if (lane == 0) {
              ct.ref[f] = ref;
              ct.kt[f] = keyed ? 1.f : __int_as_float(max(top, 1) << 23);
            }
            if (ref > 255) {
#pragma unroll
              for (int y = 0; y < KT; y += 32) {
                const int j = lane + y, e = ev[j];
                const bool nan = e == 255, in = j < left;
                ct.fk[f][j] = exp_scale(ek[j]);
                ct.ev[f][j] = nan || !in ? 0 : (uint8_t)e;
                ct.fv[f][j] = nan || !in ? 0.f : exp_scale(e);
                const uint32_t nans = __ballot_sync(0xffffffffu, nan && in);
                if (lane == 0) ct.nan[f][y >> 5] = nans;
              }
            }
          }
          convert(sm + 2 * NS * S::TILE + rs * S::RAW + (is_v ? S::RAW / 2 : 0), sm + ((is_v ? NS : 0) + st) * S::TILE, is_v ? ev : ek, top, is_v ? kUp<FMT> : 0, left);
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(smem_u32(is_v ? &ct.vfull[st] : &ct.kfull[st]));
            mbar_arrive(smem_u32(&ct.raw_empty[rs]));
          }
        } else {
          if (!(ok = warp_wait(&ct.vfull[st], cnt / NS & 1, abort_flag, g.spin))) break;
          if ((t + 1) * KT > min(p.all_see, p.n_keys)) {
            // some row does not see some key: 0 x NaN would reach it, so non-finite elements are dropped here and put
            // back at the end for the rows that do see them
            bool hit = false;
#pragma unroll 2
            for (int i = ti; i < S::TILE / 16; i += 128) {
              const uint32_t a = vbuf + st * S::TILE + i * 16;
              uint4 v = lds128(a);
              bool h = false;
              v.x = drop_nonfinite(v.x, h);
              v.y = drop_nonfinite(v.y, h);
              v.z = drop_nonfinite(v.z, h);
              v.w = drop_nonfinite(v.w, h);
              if (h) sts128(a, v);
              hit = hit || h;
            }
            if (hit) *reinterpret_cast<volatile int*>(&ct.dropped) = 1;
            fence_proxy_async_smem();
          }
          warp_arrive(&ct.vclean[st]);
        }
      }
      if (!ok) break;
      if (lane == 0) piece_free(k);
    }
    if (!ok) {
      set_status(g.status, kStatusTimeoutProducer);
      *abort_flag = 1;
    }
  } else if (warp >= 4) {
    reg_inc<160>();
    // ------------------------------------------------------------ softmax: thread = row of stream x
    const int x = (warp >> 2) - 1, r = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);         // TMEM lane quadrant of the warp
    const uint32_t tS = lanes + kColS + x * kSP, tP = lanes + kColP + x * kSP, tO = lanes + kColO + x * 128;
    int cnt0 = 0, n_s = 0, n_ml = 0;
    bool ok = true;
    struct Row {
      bool two, in;
      int row, node, head;   // of the row tile; the row's node; its query head
    };
    auto row_of = [&](const Piece& p) {
      Row w;
      w.two = p.nrows > 128;
      w.row = (w.two ? x * 128 : 0) + r;
      w.in = w.row < p.nrows;
      const int R = p.r0 + min(w.row, p.nrows - 1);
      w.node = R / g.G;
      w.head = p.h * g.G + R - w.node * g.G;
      return w;
    };
    const float scale_l2 = g.scale * 1.4426950408889634f;
    // The q rows of a piece to where the products read them: bf16 as it is, or f16 with the largest element's power of two
    // taken out (a row's softmax scale with it is returned).  A warp reads its 32 rows in 256-byte runs (D = 128) and
    // turns them, half a row at a time, through shared memory: into the operand tile of stream 1, or into the lanes'
    // rows in TMEM.
    auto put_q = [&](const Piece& p) {
      const bool two = p.nrows > 128;
      constexpr int C = D / 8, RPI = 32 / C, N = 32 / RPI;              // chunks per row, rows per load, loads
      const int row0 = (two ? x * 128 : 0) + (warp & 3) * 32 + lane / C, chunk = lane % C;
      uint4 u[N];
      int node = (p.r0 + row0) / g.G, head = p.r0 + row0 - node * g.G;  // of the row, and its head of the group
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bf16* src = q + (size_t)(p.bi.start + node) * g.ld_q + (size_t)(p.h * g.G + head) * D;
        u[i] = row0 + i * RPI < p.nrows ? reinterpret_cast<const uint4*>(src)[chunk] : make_uint4(0, 0, 0, 0);
        head += RPI;
#pragma unroll
        for (int y = 0; y < RPI; ++y)
          if (head >= g.G) head -= g.G, ++node;
      }
      float rf = scale_l2;
      if constexpr (Q8) {
        // The rows' largest elements: each step halves the lanes that hold one row and the rows that a lane holds, so
        // lane c of a row's C lanes ends with row c's.
        static_assert(N == C, "as many loads as lanes on a row");
        uint32_t amax[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
          amax[i] = 0;
#pragma unroll
          for (int y = 0; y < 4; ++y) amax[i] = max(amax[i], max(w[y] << 16 & 0x7fff0000u, w[y] & 0x7fff0000u));
        }
#pragma unroll
        for (int o = C / 2; o > 0; o >>= 1) {
          const bool up = lane & o;
#pragma unroll
          for (int i = 0; i < o; ++i) {
            const uint32_t send = up ? amax[i] : amax[i + o], keep = up ? amax[i + o] : amax[i];
            amax[i] = max(keep, __shfl_xor_sync(0xffffffffu, send, o));
          }
        }
        const int e = min(max((int)(amax[0] >> 23), 27), 227);
        const int own = __shfl_sync(0xffffffffu, e, lane % RPI * C + lane / RPI);   // of the row whose thread this is
        rf *= __int_as_float(own << 23) * kHalfUnit<FMT>;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float inv = __int_as_float((254 - __shfl_sync(0xffffffffu, e, (lane & ~(C - 1)) | i)) << 23);
          uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
          for (int y = 0; y < 4; ++y) w[y] = pack2<FMT>(__uint_as_float(w[y] << 16) * inv, __uint_as_float(w[y] & 0xffff0000u) * inv);
          u[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      const uint32_t stage = x == 0 ? qstage : qbuf;                    // [128 rows][128 B], swizzled as the operand tile is
#pragma unroll
      for (int b = 0; b < D / 64; ++b) {
        if (x == 0 || two) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int rr = (warp & 3) * 32 + i * RPI + lane / C;
            if (chunk / 8 == b) sts128(stage + (x == 0 ? 0 : b * (128 * 128)) + rr * 128 + (((chunk & 7) ^ (rr & 7)) << 4), u[i]);
          }
        }
        if (x == 0) {
          __syncwarp();
          uint32_t v[32];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint4 t = lds128(stage + r * 128 + ((i ^ (r & 7)) << 4));
            v[4 * i] = t.x, v[4 * i + 1] = t.y, v[4 * i + 2] = t.z, v[4 * i + 3] = t.w;
          }
          tmem_st32(lanes + kColQ + 32 * b, v);
          __syncwarp();
        }
      }
      if (x == 0) tmem_wait_st();
      else fence_proxy_async_smem();
      tc_fence_before();
      warp_arrive(&ct.q_ready);
      return rf;
    };
    float rf = 0.f, m = -INFINITY, l = 0.f;
    int er = 1, nt = 0;                                                 // er: 8-bit: exponent byte that the weights and O are relative to
    bool begun = false, two = false;
    // One turn: the next piece's Q goes out, then the last piece's output (its products are done, and the next one's first
    // S runs meanwhile), then the next piece's tiles.
#pragma unroll 1
    for (int piece = -1;;) {
      if (!(ok = __all_sync(0xffffffffu, piece_wait(piece + 1)))) break;
      const Piece& nxt = ct.piece[(piece + 1) % kPieces];
      const bool more = nxt.tiles != 0;
      float(&ml)[2][3][128] = ct.ml[piece & 1];
      if (piece >= 0 && !two) {
        ml[x][0][r] = m;
        ml[x][1][r] = l;
        ml[x][2][r] = begun ? (float)er : -1.f;                         // -1: the stream had no tile, its O is not there
        warp_arrive(&ct.ml_ready);
        if (!(ok = warp_wait(&ct.ml_ready, n_ml++ & 1, abort_flag, g.spin))) break;
      }
      float rf_next = 0.f;
      if (more) rf_next = put_q(nxt);
      if (piece >= 0) {
        if (!(ok = warp_wait(&ct.o_done, piece & 1, abort_flag, g.spin))) break;
        const Piece& cur = ct.piece[piece % kPieces];
        tc_fence_after();
        float f0 = 1.f, f1 = 0.f, M = m, L = l;
        int E = er;
        if (!two) {
          const float m0 = ml[0][0][r], m1 = ml[1][0][r], e0 = ml[0][2][r], e1 = ml[1][2][r];
          M = fmaxf(m0, m1);
          const float ms = M == -INFINITY ? 0.f : M;
          f0 = fast_exp2(m0 - ms), f1 = e1 < 0.f ? 0.f : fast_exp2(m1 - ms);
          L = f0 * ml[0][1][r] + (e1 < 0.f ? 0.f : f1 * ml[1][1][r]);
          if constexpr (Q8) {                                             // both relative to the larger weight x scale
            E = min(max((int)floorf(fmaxf(m0 - ms + e0, e1 < 0.f ? -INFINITY : m1 - ms + e1)), 1), 253);
            f0 = fast_exp2(m0 - ms + (e0 - (float)E));
            f1 = e1 < 0.f ? 0.f : fast_exp2(m1 - ms + (e1 - (float)E));
          }
        }
        float inv = L == 0.f ? 0.f : 1.f / L;                             // a row that sees nothing: zeros
        if constexpr (Q8) inv *= kHalfUnit<FMT> / (1 << kUp<FMT>) * __int_as_float(E << 23);
        const Row cw = row_of(cur);
        const bool join = !two && nt > 1;
        const size_t at = (size_t)(cur.bi.start + cw.node) * g.n_heads + cw.head;
        const bool to_out = sc.chunk_tiles ? cur.tiles <= sc.chunk_tiles : cur.whole();
        const size_t slot = (size_t)blockIdx.x * 2 + (cur.index ? 1 : 0);
        const size_t part = sc.chunk_tiles ? at * g.splits + cur.t0 / sc.chunk_tiles : slot * sc.rows + cw.row;
        // partial outputs: row by row for the fixed split's join; else four columns of all rows, then the next four, so
        // that a warp's store is one run of 512 bytes (row by row its 32 lines took 4 k clocks of a piece)
        float4* const po = reinterpret_cast<float4*>(g.part_o) + (sc.chunk_tiles ? part * (D / 4) : slot * (D / 4) * sc.rows + cw.row);
        const int po_step = sc.chunk_tiles ? 1 : sc.rows;
        // one row tile: each stream's threads write half of the columns
        const int d0 = two ? 0 : x * (D / 2), d1 = two ? D : d0 + D / 2;
#pragma unroll 1
        for (int d = d0; d < d1; d += 16) {
          uint32_t o[16], o1[16];
          tmem_ld_16(two ? tO + d : lanes + kColO + d, o);
          if (join) tmem_ld_16(lanes + kColO + 128 + d, o1);
          tmem_wait_ld();
          float z[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) z[j] = __uint_as_float(o[j]) * (f0 * inv);
          if (join) {
#pragma unroll
            for (int j = 0; j < 16; ++j) z[j] = fmaf(__uint_as_float(o1[j]), f1 * inv, z[j]);
          }
          if (!Q8 && cw.in && *reinterpret_cast<volatile int*>(&ct.dropped)) {   // the dropped elements of keys this row sees,
            const uint64_t* mk = g.mask ? g.mask + (size_t)(cur.bi.start + cw.node) * g.words : nullptr;
#pragma unroll 1
            for (int key = max(cur.t0 * KT, min(cur.all_see, cur.n_keys) / KT * KT); key < min(cur.t1 * KT, cur.n_keys); ++key)   // in partial tiles
              if (sees32(mk, g.words, cw.node, key - cur.bi.ctx) & 1) {
                const bf16* vp = static_cast<const bf16*>(c.v) + (cache_slot(c, cur.bi.row, cur.h, key)) * D + d;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                  const float y = __bfloat162float(vp[j]);
                  if (!(fabsf(y) < INFINITY)) z[j] += y;
                }
              }
          }
          if (cw.in && to_out) {
#pragma unroll
            for (int j = 0; j < 16; j += 8)
              *reinterpret_cast<uint4*>(out + at * D + d + j) =
                  make_uint4(pack2<EESD_KV_MODEL>(z[j], z[j + 1]), pack2<EESD_KV_MODEL>(z[j + 2], z[j + 3]),
                             pack2<EESD_KV_MODEL>(z[j + 4], z[j + 5]), pack2<EESD_KV_MODEL>(z[j + 6], z[j + 7]));
          } else if (cw.in) {
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              po[(size_t)((d + j) / 4) * po_step] = make_float4(z[j], z[j + 1], z[j + 2], z[j + 3]);
          }
          __syncwarp();
        }
        tc_fence_before();
        warp_arrive(&ct.epi_done);
        if (cw.in && !to_out && (two || x == 0)) g.part_ml[part] = make_float2(M, L);
        if (tid == 128 && !sc.chunk_tiles && cur.t0 == 0 && cur.t1 < cur.tiles)
          sc.cuts[blockIdx.x] = TcCut{cur.bi.start, cur.r0, cur.nrows, cur.h, cur.index ? 1 : 0,
                                      (int)((cur.u0 + kUnitCost + cur.tiles - 1) / ct.run)};
        cnt0 += nt;
        __syncwarp();
        if (lane == 0) piece_free(piece);
      }
      if (!more) break;
      ++piece;
      const Piece& cur = nxt;
      nt = cur.t1 - cur.t0;
      two = cur.nrows > 128;
      rf = rf_next;
      m = -INFINITY;
      l = 0.f;
      er = 1;
      begun = false;
      const int whole_to = min(cur.all_see, cur.n_keys);
#pragma unroll 1
      for (int i = two ? 0 : x; i < nt; i += two ? 1 : 2) {
        const int t = cur.t0 + i, cnt = cnt0 + i, f = cnt % FR;
        if (!(ok = warp_wait(&ct.s_full[x], n_s & 1, abort_flag, g.spin))) break;
        tc_fence_after();
        uint32_t a[KT];
        tmem_ld32(tS, a);
        tmem_ld32(tS + 32, a + 32);
        const int how = Q8 ? ct.ref[f] : 0;
        const float rt = Q8 ? rf * ct.kt[f] : rf;
        tmem_wait_ld();
        tc_fence_before();
        warp_arrive(&ct.s_free[x]);
        // the product that read the last P is done by now, most often: asked here, looked at when P is ready
        const bool pv_was_done = n_s == 0 || mbar_test_wait(smem_u32(&ct.pv_done[x]), (n_s - 1) & 1);
        const bool partial = (t + 1) * KT > whole_to;                   // some row does not see some key of the tile
        // Every choice below is made so that what a row does not see does not change a bit of its result: the forms of the
        // exponent differ between rows only by the row's own scores.
        int em = how & 255;                                             // V's largest exponent among the keys that the row sees
        if (__builtin_expect(partial || how > 255, 0)) {                // which keys those are
          if (how & kHowK) {
#pragma unroll
            for (int j = 0; j < KT; ++j) a[j] = __float_as_uint(__uint_as_float(a[j]) * ct.fk[f][j]);
          }
          const int node = row_of(cur).node, left = cur.n_keys - t * KT;
          const uint64_t* mk = g.mask ? g.mask + (size_t)(cur.bi.start + node) * g.words : nullptr;
          uint32_t s0 = sees32(mk, g.words, node, t * KT - cur.bi.ctx), s1 = sees32(mk, g.words, node, t * KT + 32 - cur.bi.ctx);
          if (left < 32) s0 &= (1u << left) - 1;
          if (left < 64) s1 &= left <= 32 ? 0u : (1u << (left - 32)) - 1;
#pragma unroll
          for (int j = 0; j < KT; ++j) a[j] = (j < 32 ? s0 : s1) >> (j & 31) & 1 ? a[j] : 0xff800000u;
          if (how & kHowV) {
            uint32_t top = 0;
#pragma unroll 2
            for (int j = 0; j < KT / 4; ++j) {
              const uint32_t bits = (j < 8 ? s0 >> 4 * j : s1 >> (4 * j - 32)) & 15;
              top = __vmaxu4(top, reinterpret_cast<const uint32_t*>(ct.ev[f])[j] & ((bits * 0x204081u & 0x1010101u) * 255u));
            }
            em = max(max(top & 255, top >> 8 & 255), max(top >> 16 & 255, top >> 24));
            if (em == 0) em = er;                                       // none: nothing that would ask for another reference
            if ((ct.nan[f][0] & s0) | (ct.nan[f][1] & s1)) l = __int_as_float(0x7fffffff);   // the row sees a V that is NaN
          }
        }
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int j = 0; j < KT; j += 4) {
          mx0 = fmaxf(mx0, fmaxf(__uint_as_float(a[j]), __uint_as_float(a[j + 1])));
          mx1 = fmaxf(mx1, fmaxf(__uint_as_float(a[j + 2]), __uint_as_float(a[j + 3])));
        }
        // O, l and m move to a new reference only when the old one is too small by 2^8, or the weights with V's scale, relative
        // to 2^er, would pass 2^12 (in range of f16).  O is then to be scaled by cf.
        // One FMA per score leaves 2^-24 |m| of it in the exponent: nothing at ordinary sizes, but at very large ones the
        // largest score has to come out as exactly 0.  V's common scale relative to er goes into the exponent, so l
        // collects the same units and is brought back by the exact power of two; beyond 2^40 weights and l go apart.
        const float mx = fmaxf(mx0, mx1) * rt, mn = fmaxf(m, mx);
        const int de = em - er;
        const bool rises = !begun || mn > m + 8.f;
        auto is_huge = [&] { return !(fabsf(m) <= 65536.f || m == -INFINITY); };
        auto is_far = [&] { return Q8 && !(how & kHowV) && abs(em - er) > 40; };
        float cf = 1.f;
        bool rescale = false, huge = false, far = false, odd = false;
        // (unless m rises or em is more than 2^3 above er, no weight passes 2^12)
        if (__builtin_expect(__any_sync(0xffffffffu, rises || is_huge() || (Q8 && (unsigned)(de + 40) > 43u)), 0)) {
          const float up = mn - m;
          float heavy = mx - mn + (float)de;                            // 8-bit: the largest weight x scale, or what it is at most: log2, over mn and 2^er
          if (__builtin_expect(how & kHowV, 0)) {                       // key by key: em may stand for a slot of no weight, and what
            heavy = -INFINITY;                                          // others see must not choose between the two forms
#pragma unroll
            for (int j = 0; j < KT; ++j)                                // (rounded as mx is)
              if (const int e = ct.ev[f][j]) heavy = fmaxf(heavy, __fadd_rn(__fmul_rn(__uint_as_float(a[j]), rt), -mn) + (float)(e - er));
          }
          const bool need = rises || (Q8 && heavy + up > 12.f);
          if (need) {
            cf = m == -INFINITY ? 0.f : fast_exp2(-up);
            l *= cf;
            if constexpr (Q8) {
              // rounded down, so that it does not creep up with every move of m; 1 .. 253 keep 2^(127 - er) a normal float
              const int en = min(max(er + (int)floorf(fmaxf(heavy, -up)), 1), 253);
              cf = m == -INFINITY ? 0.f : fast_exp2((float)(er - en) - up);
              er = en;
            }
            m = mn;
          }
          rescale = begun && __any_sync(0xffffffffu, need);
          huge = is_huge(), far = is_far();
          odd = __any_sync(0xffffffffu, huge || far);
        }
        const int dd = Q8 && !(how & kHowV) && !far ? em - er : 0;
        const float ms = m == -INFINITY ? 0.f : m, nbs = (float)dd - ms;
        const float vc = Q8 ? __int_as_float((254 - er) << 23) : 0.f;   // 2^(127 - er)
        uint32_t w[KT / 2];
        f32x2 sum0 = pack_f2(0.f, 0.f), sum1 = pack_f2(0.f, 0.f);
        if (__builtin_expect(!odd, 1)) {
          const f32x2 nb = pack_f2(nbs, nbs), rt2 = pack_f2(rt, rt);
          if (__builtin_expect(!(how & kHowV), 1)) {
#pragma unroll
            for (int j = 0; j < KT; j += 4) {
              const float2 y0 = unpack_f2(fma2(pack_f2(__uint_as_float(a[j]), __uint_as_float(a[j + 1])), rt2, nb));
              const float2 y1 = unpack_f2(fma2(pack_f2(__uint_as_float(a[j + 2]), __uint_as_float(a[j + 3])), rt2, nb));
              const float e0 = fast_exp2(y0.x), e1 = fast_exp2(y0.y), e2 = fast_exp2(y1.x), e3 = fast_exp2(y1.y);
              sum0 = add2(sum0, pack_f2(e0, e1));
              sum1 = add2(sum1, pack_f2(e2, e3));
              w[j / 2] = pack2<FMT>(e0, e1);
              w[j / 2 + 1] = pack2<FMT>(e2, e3);
            }
          } else {
#pragma unroll
            for (int j = 0; j < KT; j += 4) {
              const float2 y0 = unpack_f2(fma2(pack_f2(__uint_as_float(a[j]), __uint_as_float(a[j + 1])), rt2, nb));
              const float2 y1 = unpack_f2(fma2(pack_f2(__uint_as_float(a[j + 2]), __uint_as_float(a[j + 3])), rt2, nb));
              const float e0 = fast_exp2(y0.x), e1 = fast_exp2(y0.y), e2 = fast_exp2(y1.x), e3 = fast_exp2(y1.y);
              const float4 v = reinterpret_cast<const float4*>(ct.fv[f])[j / 4];
              sum0 = add2(sum0, pack_f2(e0, e1));
              sum1 = add2(sum1, pack_f2(e2, e3));
              // an unseen key's factor may be out of range, its weight is 0
              w[j / 2] = pack2<FMT>(e0 == 0.f ? 0.f : e0 * v.x * vc, e1 == 0.f ? 0.f : e1 * v.y * vc);
              w[j / 2 + 1] = pack2<FMT>(e2 == 0.f ? 0.f : e2 * v.z * vc, e3 == 0.f ? 0.f : e3 * v.w * vc);
            }
          }
        } else {                                                        // the same, row by row in its own form
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < KT; j += 2) {
            float e[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const float y = __uint_as_float(a[j + b]);
              const float z = huge ? __fadd_rn(__fadd_rn(__fmul_rn(y, rt), -ms), (float)dd) : fmaf(y, rt, nbs);
              e[b] = fast_exp2(z);
              sum[(j + b) & 3] += e[b];
              if (how & kHowV) e[b] = e[b] == 0.f ? 0.f : e[b] * ct.fv[f][j + b] * vc;
              if (far) e[b] = fast_exp2(z + (float)(em - er));
            }
            w[j / 2] = pack2<FMT>(e[0], e[1]);
          }
          sum0 = pack_f2(sum[0], sum[1]);
          sum1 = pack_f2(sum[2], sum[3]);
        }
        const float2 sv = unpack_f2(add2(sum0, sum1));
        l = Q8 ? fmaf(sv.x + sv.y, __int_as_float((127 - dd) << 23), l) : l + (sv.x + sv.y);
        // ---- P, once the product that read the last one is done (O is at rest then)
        if (!__all_sync(0xffffffffu, pv_was_done) && !(ok = warp_wait(&ct.pv_done[x], (n_s - 1) & 1, abort_flag, g.spin))) break;
        ++n_s;
        tc_fence_after();
        if (__builtin_expect(rescale, 0)) {
#pragma unroll 1
          for (int b = 0; b < D; b += 16) {
            uint32_t o[16];
            tmem_ld_16(tO + b, o);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * cf);
            tmem_st_16(tO + b, o);
          }
        }
        // the other stream's threads may still read this stream's O of the piece before
        if (__builtin_expect(!begun, 0) && piece && !(ok = warp_wait(&ct.epi_done, (piece - 1) & 1, abort_flag, g.spin))) break;
        begun = true;
        tmem_st32(tP, w);
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(&ct.p_ready[x]);
      }
      if (!ok) break;
    }
    if (!ok) {
      set_status(g.status, kStatusTimeoutEpilogue);
      *abort_flag = 1;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// Joins the pieces of the unit that goes from run blockIdx.x on into the next ones, in run order.  A block has 32 rows and
// 64 columns, a lane one row and a warp 16 columns.  Bound by the latency of its loads where a unit is in many pieces (a
// long context of one KV head: all of them), so the warps share the search for the largest reference and four pieces'
// loads are in flight (two blocks of one KV head at up to 66 k slots, 60 pieces a unit: 112 -> 52 us in all).
template <int D>
__global__ void __launch_bounds__(128) attn_tree_tc_join_kernel(TreeGeom g, TcSchedule sc, bf16* __restrict__ out) {
  pdl_trigger();
  pdl_wait();
  constexpr int W = 4, U = 4, N = 16;
  __shared__ float top[W][32];
  const int c0 = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = (blockIdx.z * W + warp) * N;
  const TcCut cut = sc.cuts[c0];
  if ((int)blockIdx.y * 32 >= cut.nrows) return;
  const int row = blockIdx.y * 32 + lane, at = min(row, cut.nrows - 1);
  auto slot = [&](int k) { return (size_t)k * 2 + (k == c0 ? cut.second : 0); };
  float M = -INFINITY, L = 0.f, acc[N];
#pragma unroll 4
  for (int k = c0 + warp; k <= cut.last; k += W) M = fmaxf(M, g.part_ml[slot(k) * sc.rows + at].x);
  top[warp][lane] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) M = fmaxf(M, top[w][lane]);
  const float ms = M == -INFINITY ? 0.f : M;
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
  for (int k0 = c0; k0 <= cut.last; k0 += U) {
    float2 ml[U];
    float4 v[U][N / 4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k0 + u > cut.last) break;
      ml[u] = g.part_ml[slot(k0 + u) * sc.rows + at];
      const float4* src = reinterpret_cast<const float4*>(g.part_o) + (slot(k0 + u) * (D / 4) + d / 4) * sc.rows + at;
#pragma unroll
      for (int j = 0; j < N / 4; ++j) v[u][j] = src[(size_t)j * sc.rows];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k0 + u > cut.last) break;
      const float w = ml[u].y * fast_exp2(ml[u].x - ms);
      L += w;
#pragma unroll
      for (int j = 0; j < N / 4; ++j) {
        acc[4 * j] = fmaf(w, v[u][j].x, acc[4 * j]);
        acc[4 * j + 1] = fmaf(w, v[u][j].y, acc[4 * j + 1]);
        acc[4 * j + 2] = fmaf(w, v[u][j].z, acc[4 * j + 2]);
        acc[4 * j + 3] = fmaf(w, v[u][j].w, acc[4 * j + 3]);
      }
    }
  }
  if (row >= cut.nrows) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int R = cut.r0 + row, node = R / g.G;
  bf16* dst = out + ((size_t)(cut.start + node) * g.n_heads + cut.h * g.G + R - node * g.G) * D + d;
  uint32_t w[N / 2];
#pragma unroll
  for (int j = 0; j < N / 2; ++j) w[j] = pack2<EESD_KV_MODEL>(acc[2 * j] * inv, acc[2 * j + 1] * inv);
#pragma unroll
  for (int j = 0; j < N / 2; j += 4) *reinterpret_cast<uint4*>(dst + 2 * j) = make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
}

template <int D, int FMT>
cudaError_t launch(const TcSchedule& sc, const TreeGeom& g, const CacheGeom& c, const CUtensorMap& km, const CUtensorMap& vm,
                   const void* q, void* out, cudaStream_t s) {
  using S = TcShape<D, FMT>;
  auto kernel = attn_tree_tc_kernel<D, FMT>;
  static SmemOnce once;
  cudaError_t e = once.set(reinterpret_cast<const void*>(kernel), S::smem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(kernel, dim3(sc.ctas), dim3(kThreads), S::smem, s, km, vm, g, c, sc, static_cast<const bf16*>(q), static_cast<bf16*>(out));
  if (e == cudaSuccess && !sc.chunk_tiles && sc.ctas > 1)
    e = launch_pdl(attn_tree_tc_join_kernel<D>, dim3(sc.ctas, (std::min(sc.rows, g.max_nodes * g.G) + 31) / 32, D / 64), dim3(128), 0, s, g, sc,
                   static_cast<bf16*>(out));
  return e;
}

}  // namespace

cudaError_t launch_attn_tree_tc(int fmt, int D, const TcSchedule& sc, const TreeGeom& g, const CacheGeom& c, const CUtensorMap& km,
                                const CUtensorMap& vm, const void* q, void* out, cudaStream_t s) {
  switch (fmt * 2 + (D == 128)) {
    case 0: return launch<64, EESD_KV_MODEL>(sc, g, c, km, vm, q, out, s);
    case 1: return launch<128, EESD_KV_MODEL>(sc, g, c, km, vm, q, out, s);
    case 2: return launch<64, EESD_KV_E4M3>(sc, g, c, km, vm, q, out, s);
    case 3: return launch<128, EESD_KV_E4M3>(sc, g, c, km, vm, q, out, s);
    case 4: return launch<64, EESD_KV_INT8>(sc, g, c, km, vm, q, out, s);
    default: return launch<128, EESD_KV_INT8>(sc, g, c, km, vm, q, out, s);
  }
}

}  // namespace eesd
