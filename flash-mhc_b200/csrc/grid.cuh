// Grid and shared-memory set-up of the persistent streaming kernels.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <mutex>
#include <new>
#include <vector>

namespace fmhc {

// Resident blocks per SM of `kernel` and the SM count, cached for the process
// (occupancy queries and attribute reads stay out of CUDA-graph captures and
// out of the per-launch cost).  T units of work, one per warp.
template <class K>
int grid_for(K kernel, int64_t T, int threads) {
  struct Entry {
    const void *k;
    int dev, per_sm, sms;
  };
  static std::mutex mu;
  static Entry cache[64];
  static int used = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  int per_sm = 0, sms = 0;
  {
    std::lock_guard<std::mutex> lock(mu);
    for (int i = 0; i < used; ++i)
      if (cache[i].k == reinterpret_cast<const void *>(kernel) && cache[i].dev == dev) {
        per_sm = cache[i].per_sm;
        sms = cache[i].sms;
      }
    if (sms == 0) {
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0);
      if (per_sm < 1) per_sm = 1;
      if (used < 64) cache[used++] = Entry{reinterpret_cast<const void *>(kernel), dev, per_sm, sms};
    }
  }
  const int64_t warps_per_block = threads / 32;
  const int64_t need = (T + warps_per_block - 1) / warps_per_block;
  const int64_t cap = int64_t(sms) * per_sm;
  return int(need < cap ? need : cap);
}

inline int sm_count() {
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms > 0 ? sms : 1;
}

constexpr size_t kMaxSmem = 232448 - 1024;  // dynamic shared memory beside a little static

// Dynamic shared memory beyond the default needs an attribute of the kernel.  Per
// kernel and device it only ever grows: another thread may be between setting it
// and its launch.
inline void allow_smem(const void *kernel, size_t bytes) {
  struct Entry {
    const void *k;
    int dev;
    size_t bytes;
  };
  static std::mutex mu;
  static std::vector<Entry> set;
  if (bytes <= 40 * 1024) return;  // beside the static arrays, below the default 48 KiB
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  auto at = std::find_if(set.begin(), set.end(), [&](const Entry &e) { return e.k == kernel && e.dev == dev; });
  if (at == set.end()) {
    try {
      at = set.insert(at, Entry{kernel, dev, 0});
    } catch (const std::bad_alloc &) {
      return;  // no exception crosses the C ABI; the launch reports its limit
    }
  }
  if (at->bytes >= bytes) return;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)) == cudaSuccess)
    at->bytes = bytes;
}

}  // namespace fmhc
