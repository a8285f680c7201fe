// capi.cu -- error reporting and version entry points of the kb200 C ABI.
#include <cstdarg>
#include <cstdio>
#include "kb200_internal.h"

namespace kb {
static thread_local char g_err[512] = "";

int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int allow_smem(const void* kernel, size_t bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e == cudaSuccess && (done.load(std::memory_order_relaxed) & bit)) return KB200_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(KB200_ERR_LAUNCH, "shared memory of %zu bytes: %s", bytes, cudaGetErrorString(e));
  }
  done.fetch_or(bit, std::memory_order_relaxed);
  return KB200_OK;
}

int sm_count() {
  static std::atomic<int> counts[64];   // per device
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return n; }
  if (dev < 64 && counts[dev]) return counts[dev];
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  if (dev < 64) counts[dev] = n;
  return n;
}

int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return set_error(KB200_ERR_LAUNCH, "%s: %s", what, cudaGetErrorString(e));
  return KB200_OK;
}
}  // namespace kb

extern "C" int kb200_abi_version(void) { return 2; }
extern "C" const char* kb200_last_error(void) { return kb::g_err; }
