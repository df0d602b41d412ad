// Facts of a device and settings of a kernel, asked or made once per device (a small call's host time counts). Host code
// only. Any number of threads, each with a current device of its own: what is shared are the flags, never the device.
#pragma once

#include <cuda_runtime_api.h>

#include <atomic>

namespace muse {

constexpr int MAX_DEVICES = 64;

// The calling thread's device, -1 where it is not known or beyond the flags.
inline int device_slot() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < MAX_DEVICES ? dev : -1;
}

inline int device_sms() {
  static std::atomic<int> sms[MAX_DEVICES];
  const int dev = device_slot();
  if (dev < 0) return 0;
  int v = sms[dev].load(std::memory_order_relaxed);
  if (v == 0) {
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    sms[dev].store(v, std::memory_order_relaxed);
  }
  return v;
}

struct DeviceOnce {
  std::atomic<bool> was[MAX_DEVICES] = {};
  // Calls `set` unless it has succeeded on the current device before. (Two threads that come first together both call it.)
  template <typename F>
  cudaError_t run(F&& set) {
    const int dev = device_slot();
    if (dev >= 0 && was[dev].load(std::memory_order_acquire)) return cudaSuccess;
    const cudaError_t e = set();
    if (e == cudaSuccess && dev >= 0) was[dev].store(true, std::memory_order_release);
    return e;
  }
};

}  // namespace muse
