// What host code has found out about a device, or set on it, once: a number of SMs, how many clusters are resident, a kernel's attributes. All of it holds for one device alone, and a process may
// have backends of several, so it is kept for each (asking which one is current costs 30 ns a launch). Threads that come to the same entry at once write the same value.
#pragma once
#include <cuda_runtime.h>

namespace mtb {

template <typename T>
struct PerDevice {
  static constexpr int MOST = 64;   // of devices that are remembered; others are asked each time
  T known[MOST] = {};
  // The current device's entry, as new before its first use.
  T& here() {
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < MOST) return known[dev];
    static thread_local T other;
    return other = T();
  }
};

// SMs of the current device.
inline int sms_here() {
  static PerDevice<int> known;
  int& n = known.here();
  if (n == 0) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) { cudaGetLastError(); n = 148; }
  }
  return n;
}

}  // namespace mtb
