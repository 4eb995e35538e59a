// host_util.h — host helpers shared by the translation units of libqora_cuda.so: the
// thread's last error message and the status-returning check macros.
#pragma once

#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <string>

#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include "../../include/qora_cuda.h"

namespace qora {

inline thread_local std::string g_last_error;

inline qora_status fail(qora_status st, const char* fmt, ...) {
  char buf[1024];
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return st;
}

inline int sm_count(int dev) {
  int n = 0;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (no libcuda link)
inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

}  // namespace qora

#define QCUDA(call)                                                                   \
  do {                                                                                \
    cudaError_t e_ = (call);                                                          \
    if (e_ != cudaSuccess)                                                            \
      return qora::fail(e_ == cudaErrorMemoryAllocation ? QORA_ERR_OOM : QORA_ERR_CUDA, \
                        "%s failed: %s (%s:%d)", #call, cudaGetErrorString(e_), __FILE__, __LINE__); \
  } while (0)

#define QCHECK(expr)                 \
  do {                               \
    qora_status s_ = (expr);         \
    if (s_ != QORA_OK) return s_;    \
  } while (0)
