// Something that is done once on every GPU of the process: a kernel's attributes belong to the device that is current.
#pragma once

#include <atomic>

#include <cuda_runtime.h>

namespace vo {

struct PerDevice {
  std::atomic<unsigned long long> done{0};  // a bit per device
  // set() on the current device unless it has succeeded there before (devices from 64 on: every time)
  template <typename F>
  cudaError_t operator()(F set) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    e = set();
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
  }
};

}  // namespace vo
