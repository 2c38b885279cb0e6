// Host-side helpers shared by the C ABI's translation units: the last-error
// message, launch checks, shared-memory limits and device queries.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <string>

#include "../../include/shrimp_b200.h"

namespace sb {

// One message per host thread for the whole library (sb_last_error).
inline thread_local std::string g_last_error;

inline int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}

// SHRIMP_B200_SYNC_DEBUG=1: synchronise and log after every launch (debugging
// aid; never set in serving).
inline bool sync_debug() {
  static const bool v = [] {  // read once (thread-safe static initialisation)
    const char* e = getenv("SHRIMP_B200_SYNC_DEBUG");
    return e && e[0] == '1';
  }();
  return v;
}

inline int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && sync_debug()) {
    fprintf(stderr, "[sb] launched %s ...", what);
    fflush(stderr);
    e = cudaDeviceSynchronize();
    fprintf(stderr, " done (%s)\n", cudaGetErrorString(e));
  }
  if (e != cudaSuccess) return fail(SB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return SB_OK;
}

inline long long cdiv(long long a, long long b) { return (a + b - 1) / b; }
inline int round_up(int a, int b) { return (a + b - 1) / b * b; }

// Raise a kernel's dynamic shared-memory limit once per (device, kernel).
inline int ensure_smem(const void* fn, int bytes) {
  struct Entry { const void* fn; int dev; int bytes; };
  static thread_local Entry cache[128];
  static thread_local int used = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  for (int i = 0; i < used; ++i)
    if (cache[i].fn == fn && cache[i].dev == dev && cache[i].bytes >= bytes) return SB_OK;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(SB_ERR_CUDA, "shared-memory attribute: %s", cudaGetErrorString(e));
  if (used < 128) cache[used++] = Entry{fn, dev, bytes};
  return SB_OK;
}

inline int num_sms() {
  // per device; host threads racing on a first query store the same value
  static std::atomic<int> cache[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) dev = 0;
  int n = cache[dev].load(std::memory_order_relaxed);
  if (!n) {
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (n <= 0) n = 148;
    cache[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace sb
