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

// Raise a kernel's dynamic shared-memory limit to `bytes` on the current device
// unless it is that high already. The limit belongs to the device's kernel, not
// to the calling thread: one table serves all host threads and never lowers it.
inline int ensure_smem(const void* fn, int bytes) {
  struct Entry { const void* fn; int dev; int bytes; };
  constexpr int kEntries = 1024;  // open addressing; more than the library has kernels
  static Entry table[kEntries];
  static std::atomic_flag lock = ATOMIC_FLAG_INIT;
  int dev = 0;
  cudaGetDevice(&dev);
  unsigned at = (unsigned)(((uintptr_t)fn >> 4) * 2654435761u + (unsigned)dev) % kEntries;
  while (lock.test_and_set(std::memory_order_acquire)) {
  }
  Entry* e = nullptr;
  for (int i = 0; i < kEntries && !e; ++i, at = (at + 1) % kEntries)
    if (!table[at].fn || (table[at].fn == fn && table[at].dev == dev)) e = &table[at];
  cudaError_t err = cudaSuccess;
  if (!e || e->fn != fn || e->bytes < bytes) {
    cudaFuncAttributes now{};
    err = cudaFuncGetAttributes(&now, fn);
    if (err == cudaSuccess && now.maxDynamicSharedSizeBytes < bytes)
      err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err == cudaSuccess && e)
      *e = Entry{fn, dev, bytes > now.maxDynamicSharedSizeBytes ? bytes : now.maxDynamicSharedSizeBytes};
  }
  lock.clear(std::memory_order_release);
  if (err != cudaSuccess) return fail(SB_ERR_CUDA, "shared-memory attribute: %s", cudaGetErrorString(err));
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
