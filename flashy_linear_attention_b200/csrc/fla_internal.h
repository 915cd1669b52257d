// What the translation units of the library share: the launch counter behind
// fla_sm100_last_launch_count(), the check of the current device and the description of failed
// calls on stderr (FLA_DEBUG=1).
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdio>
#include <cstdlib>

#include "../../include/flashlinear_sm100.h"

namespace fla {

extern thread_local int g_last_launches;  // kernels launched by the last call on this thread

inline bool describe_failures() {
  static const bool on = [] {
    const char* e = getenv("FLA_DEBUG");
    return e != nullptr && e[0] == '1';
  }();
  return on;
}

// FLA_OK on an sm_100 device; its number of SMs.
inline int block_device(int* sm_count) {
  static std::atomic<int> sms[64];  // 0: not asked yet, -1: another architecture
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return FLA_ERR_CUDA;
  int n = sms[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    int major = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return FLA_ERR_CUDA;
    if (major != 10) n = -1;
    sms[dev].store(n, std::memory_order_relaxed);
  }
  if (n < 0) return FLA_ERR_DEVICE;
  *sm_count = n;
  return FLA_OK;
}

inline int launched(cudaError_t e, const char* kernel) {
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e == cudaSuccess) {
    ++g_last_launches;
    return FLA_OK;
  }
  (void)cudaGetLastError();
  if (describe_failures()) fprintf(stderr, "[flashlinear_sm100] launch of %s failed: %s\n", kernel, cudaGetErrorString(e));
  return FLA_ERR_CUDA;
}

}  // namespace fla
