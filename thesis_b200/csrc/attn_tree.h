// Internal interface of the tree attention and its C entry points' helpers (not part of the C ABI).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "../../include/eesd.h"

namespace eesd {

struct CacheGeom;

// The dynamic shared memory limit of one kernel, raised once per device.
struct SmemOnce {
  std::atomic<uint64_t> done{0};   // bit: device
  cudaError_t set(const void* kernel, size_t bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
  }
};

// record a formatted message for eesd_last_error() and return `code`
int fail_arg(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
// the stream must be one of the current device's (a launch on another device's stream would read foreign memory)
int check_stream(const char* who, void* stream);
int check_cache(const char* who, int dtype, const EesdKvCache* c, int layer);
int check_tree(const char* who, const EesdTree* t);
CacheGeom cache_layer(const EesdKvCache* c, int dtype, int layer);
inline size_t cache_elem_bytes(const EesdKvCache* c, int dtype) {
  return c->format != EESD_KV_MODEL ? 1 : dtype == EESD_BF16 ? 2 : 4;
}

}  // namespace eesd
