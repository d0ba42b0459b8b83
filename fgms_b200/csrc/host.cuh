// What the host code of every entry point uses: errors, launches that are counted, the device, ranges of memory.  One of each for the whole
// library, whichever source file an entry point is in.
#pragma once
#include "../../include/fgms_b200.h"

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>

#include <nvtx3/nvToolsExt.h>

namespace fgms_host {

inline thread_local char g_err[512] = "";
inline std::atomic<long long> g_launches{0};
// launches that the shape alone would have sent to the tensor-core kernels but that ran on the CUDA-core
// kernels (base pointers not 16-byte aligned): fgms_b200_fallback_count()
inline std::atomic<long long> g_fallbacks{0};
// SMs the persistent kernels leave free (fgms_b200_set_reserved_sms): room for a kernel of another stream
inline std::atomic<int> g_reserved_sms{0};

inline int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

inline int check_launch(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(FGMS_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return FGMS_OK;
}

struct DeviceInfo {
  int sms = 0;       // to launch on
  int reserved = 0;  // to leave free
  int max_smem_optin = 0;
};

inline int device_info(DeviceInfo* out) {
  static thread_local int cached_dev = -1;
  static thread_local DeviceInfo cached;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return fail(FGMS_ERR_CUDA, "cudaGetDevice: %s", cudaGetErrorString(e));
  if (dev != cached_dev) {
    cudaDeviceProp prop;
    e = cudaGetDeviceProperties(&prop, dev);
    if (e != cudaSuccess) return fail(FGMS_ERR_CUDA, "cudaGetDeviceProperties: %s", cudaGetErrorString(e));
    cached.sms = prop.multiProcessorCount;
    cached.max_smem_optin = (int)prop.sharedMemPerBlockOptin;
    cached_dev = dev;
  }
  *out = cached;
  const int keep = g_reserved_sms.load(std::memory_order_relaxed);
  out->reserved = keep;
  if (keep > 0) out->sms = cached.sms - keep > 1 ? cached.sms - keep : 1;
  return FGMS_OK;
}

// NVTX range named after the entry point, open for the duration of the host call (the enqueue); a timeline tool
// shows the kernels launched inside it under that name.  Without a tool attached the calls return at once.
struct TraceRange {
  explicit TraceRange(const char* name) { nvtxRangePushA(name); }
  ~TraceRange() { nvtxRangePop(); }
  TraceRange(const TraceRange&) = delete;
  TraceRange& operator=(const TraceRange&) = delete;
};

struct Range {
  const void* p;
  size_t bytes;
  bool overlaps(const Range& o) const {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(o.p);
    return a < b + o.bytes && b < a + bytes;
  }
};

// Adds a source file's count of problems on the current device (each has its own: device code is linked file by file), and clears it.
inline int take_problems(const unsigned long long& counter, int reset, unsigned long long* sum) {
  unsigned long long v = 0;
  const unsigned long long zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, counter, sizeof(v));
  if (e == cudaSuccess && reset) e = cudaMemcpyToSymbol(counter, &zero, sizeof(zero));
  if (e != cudaSuccess) return fail(FGMS_ERR_CUDA, "the count of problems: %s", cudaGetErrorString(e));
  *sum += v;
  return FGMS_OK;
}
int take_layer_problems(int reset, unsigned long long* sum);  // of layers_abi.cu

}  // namespace fgms_host
