// More than 64 KB of LDS for a kernel: allowed once a device. (The HIP runtime's header comes before this one.)
#pragma once
#include <stdint.h>

#include <atomic>

struct KernelLds {
  const void *kern;
  int bytes;
};
// done: a bit for each of the first 64 devices, of these kernels; on a device past them they are allowed at each call
template <int N>
hipError_t allow_lds_once(const KernelLds (&k)[N], std::atomic<uint64_t> &done) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
  if (done.load() & bit) return hipSuccess;
  for (const KernelLds &x : k) {
    e = hipFuncSetAttribute(x.kern, hipFuncAttributeMaxDynamicSharedMemorySize, x.bytes);
    if (e != hipSuccess) return e;
  }
  done |= bit;
  return hipSuccess;
}
inline hipError_t allow_lds_once(const void *kern, int bytes, std::atomic<uint64_t> &done) {
  const KernelLds k[] = {{kern, bytes}};
  return allow_lds_once(k, done);
}
