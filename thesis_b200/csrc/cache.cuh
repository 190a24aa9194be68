// KV cache in the model dtype or in 8 bits: geometry, exponents and conversions shared by the append,
// read, compaction and attention kernels of the tree-draft path.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace eesd {

// One layer of an EesdKvCache as the kernels see it.
struct CacheGeom {
  int n_kv_heads, max_batch, max_seq;
  const void* k;
  const void* v;
  const uint8_t* ke;   // exponent bytes [max_batch, Hkv, max_seq], 8-bit formats only
  const uint8_t* ve;
};

// element offset of (row, head, slot): 64-bit, a long cache passes 2^31 elements
__device__ __forceinline__ size_t cache_slot(const CacheGeom& c, int row, int head, int slot) {
  return ((size_t)row * c.n_kv_heads + head) * c.max_seq + slot;
}

// Exponent byte of a vector whose largest |x| has the bit pattern `amax` (|x| ordered as uint, so NaN and
// infinity come out on top): 255 for those, else e + 127 with e the smallest integer >= -100 with
// amax <= Q 2^e.  Q = 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6: comparing the mantissa decides exactly.
template <int FMT> __device__ __forceinline__ int exp_byte(uint32_t amax) {
  if (amax >= 0x7f800000u) return 255;
  constexpr int kShift = FMT == EESD_KV_E4M3 ? 8 : 6;
  constexpr uint32_t kMant = FMT == EESD_KV_E4M3 ? 0x600000u : 0x7e0000u;
  const int x = (int)(amax >> 23) - 127;
  const int e = x - kShift + ((amax & 0x7fffffu) > kMant ? 1 : 0);
  return max(e, -100) + 127;
}
// 2^e and 2^-e from the byte (27 .. 249: both are normal floats); a 255 byte reads back as NaN
__device__ __forceinline__ float exp_scale(int byte) {
  return byte == 255 ? __int_as_float(0x7fffffff) : __int_as_float(byte << 23);
}
__device__ __forceinline__ float exp_inv_scale(int byte) { return byte == 255 ? 0.f : __int_as_float((254 - byte) << 23); }

// two elements -> two bytes (a in the low one); the arguments are already scaled into the format's range
template <int FMT> __device__ __forceinline__ uint32_t quant2(float a, float b) {
  if constexpr (FMT == EESD_KV_E4M3) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
  } else {
    return (uint32_t)(__float2int_rn(a) & 255) | ((uint32_t)(__float2int_rn(b) & 255) << 8);
  }
}

// Bytes -> halves without conversion instructions.  Input: four stored bytes in `w`; output: bytes 0, 1 in
// `lo` and 2, 3 in `hi`, as f16 pairs holding the element times 2^-8 (e4m3: its sign, exponent and mantissa
// bits moved under an f16 exponent whose bias is 8 larger, subnormals included) or the element itself (int8:
// 0x6400 + u is 1024 + u exactly, u = element + 128).  Both are exact.
template <int FMT> __device__ __forceinline__ uint32_t bytes_to_half2(uint32_t placed) {
  if constexpr (FMT == EESD_KV_E4M3) {
    return ((placed >> 1) & 0x3f803f80u) | (placed & 0x80008000u);      // bytes sit in the high half of each lane
  } else {
    const __half2 k = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));   // 1152
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&placed), k);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <int FMT> __device__ __forceinline__ void unpack4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == EESD_KV_E4M3) {
    lo = bytes_to_half2<FMT>(__byte_perm(w, 0, 0x1404));   // [0 | b0 << 8, 0 | b1 << 8]
    hi = bytes_to_half2<FMT>(__byte_perm(w, 0, 0x3424));
  } else {
    w ^= 0x80808080u;
    lo = bytes_to_half2<FMT>(__byte_perm(w, 0x64646464u, 0x4140));
    hi = bytes_to_half2<FMT>(__byte_perm(w, 0x64646464u, 0x4342));
  }
}
// factor between unpack4's halves and the element
template <int FMT> constexpr float kHalfUnit = FMT == EESD_KV_E4M3 ? 256.f : 1.f;

__device__ __forceinline__ float2 half2_to_float2(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

}  // namespace eesd
