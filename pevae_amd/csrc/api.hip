// Error reporting and device queries of libpevae_hip.so.
#include "common.h"
#include "../../include/pevae_hip.h"
#include <stdarg.h>
#include <string.h>

static thread_local char g_err[512] = "";

void pv_set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
}

template <class T>
static __global__ __launch_bounds__(256) void clear_kernel(T* __restrict__ p, size_t n) {
  for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < n; i += gridDim.x * (size_t)256) p[i] = T{};
}
template <class T>
static void launch_clear(void* p, size_t bytes, hipStream_t stream) {
  const size_t n = bytes / sizeof(T), want = (n + 255) / 256;
  clear_kernel<T><<<dim3((unsigned)(want > 4096 ? 4096 : want)), dim3(256), 0, stream>>>((T*)p, n);
}
int pv_clear(void* p, size_t bytes, hipStream_t stream) {
  PV_REQUIRE(p && bytes % 4 == 0 && ((uintptr_t)p & 3) == 0, "pv_clear: not a number of 4-byte words");
  if (bytes == 0) return PV_OK;
  if (((uintptr_t)p & 15) == 0 && bytes % 16 == 0)
    launch_clear<uint4>(p, bytes, stream);
  else
    launch_clear<uint32_t>(p, bytes, stream);
  PV_LAUNCH_CHECK("clear_kernel");
  return PV_OK;
}

extern "C" {

const char* pv_last_error(void) { return g_err; }

int pv_abi_version(void) { return PV_ABI_VERSION; }

int pv_device_info(int* cu_count, int* lds_bytes, char* arch, int arch_len) {
  int dev = 0;
  PV_HIP(hipGetDevice(&dev));
  hipDeviceProp_t prop;
  PV_HIP(hipGetDeviceProperties(&prop, dev));
  if (cu_count) *cu_count = prop.multiProcessorCount;
  if (lds_bytes) *lds_bytes = (int)prop.maxSharedMemoryPerMultiProcessor;
  if (arch && arch_len > 0) {
    strncpy(arch, prop.gcnArchName, arch_len - 1);
    arch[arch_len - 1] = 0;
  }
  return PV_OK;
}

}  // extern "C"
