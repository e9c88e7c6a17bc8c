// csrc/lds_once.h over a HIP runtime of three functions: what it sets, for which device.
typedef int hipError_t;
constexpr int hipSuccess = 0, hipFuncAttributeMaxDynamicSharedMemorySize = 8;
static int g_dev, g_fail, g_sets, g_bytes[128][2];
static hipError_t hipGetDevice(int *d) {
  *d = g_dev;
  return hipSuccess;
}
static hipError_t hipFuncSetAttribute(const void *f, int, int bytes) {
  if (g_fail) return 7;
  g_sets++;
  g_bytes[g_dev][f != nullptr] = bytes;
  return hipSuccess;
}
#include "../hexanima_amd/csrc/lds_once.h"

extern "C" int host_allow(int dev, int fail) {
  static std::atomic<uint64_t> done{0};
  g_dev = dev;
  g_fail = fail;
  const KernelLds k[] = {{nullptr, 100}, {&g_dev, 200}};
  return allow_lds_once(k, done);
}
extern "C" int host_sets() { return g_sets; }
extern "C" int host_bytes(int dev, int which) { return g_bytes[dev][which]; }
