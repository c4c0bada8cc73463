// dkv_launch.h — host-side launch helpers that remember per device what costs a driver call to ask or to set.
#pragma once
#include <atomic>
#include <cstdint>
#include <cuda_runtime.h>

namespace dkv {

// SMs of the current device.
inline int device_sms() {
  static std::atomic<int> known[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev < 64 && known[dev].load(std::memory_order_relaxed) > 0) return known[dev].load(std::memory_order_relaxed);
  int sms = 148;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  if (dev < 64) known[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

// Lets `kernel` use `bytes` of dynamic shared memory on the current device; `done` remembers the devices.
template <typename Kernel>
bool allow_shared(Kernel kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;
  if (done.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

}  // namespace dkv
