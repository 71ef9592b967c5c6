// capi_internal.h — shared plumbing of the C ABI implementation (host side).
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "../../include/hxm.h"

namespace hxm {

// Thread-local last-error message (returned by hxm_last_error_string()).
void set_error(const char* fmt, ...);
void clear_error();

// Returns HXM_ECUDA (with the message recorded) if the last launch failed.
hxm_status check_launch(const char* what);

inline size_t dtype_size(hxm_dtype t) { return t == HXM_F32 ? 4 : 2; }

}  // namespace hxm

#define HXM_REQUIRE(cond, ...)          \
  do {                                  \
    if (!(cond)) {                      \
      ::hxm::set_error(__VA_ARGS__);    \
      return HXM_EBADARG;               \
    }                                   \
  } while (0)

#define HXM_REQUIRE_SUPPORTED(cond, ...) \
  do {                                   \
    if (!(cond)) {                       \
      ::hxm::set_error(__VA_ARGS__);     \
      return HXM_EUNSUPPORTED;           \
    }                                    \
  } while (0)

#define HXM_CUDA_TRY(expr)                                                              \
  do {                                                                                  \
    cudaError_t e_ = (expr);                                                            \
    if (e_ != cudaSuccess) {                                                            \
      ::hxm::set_error("%s failed: %s", #expr, cudaGetErrorString(e_));                 \
      return HXM_ECUDA;                                                                 \
    }                                                                                   \
  } while (0)

namespace hxm {

// Lets Kernel use all of the shared memory that a block can have, once per device.  A limit of each call's own size
// could be lowered by another thread's call before the launch, which is refused then.  kPreferShared: an SM's
// memory goes to shared memory as far as it can, for as many blocks as fit.
template <auto Kernel, bool kPreferShared = false>
inline hxm_status allow_shared_memory() {
  static std::atomic<unsigned long long> done{0};  // a bit per device
  int dev = 0;
  HXM_CUDA_TRY(cudaGetDevice(&dev));
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return HXM_OK;
  int most = 0;
  cudaFuncAttributes at{};
  HXM_CUDA_TRY(cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev));
  HXM_CUDA_TRY(cudaFuncGetAttributes(&at, Kernel));
  HXM_CUDA_TRY(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most - (int)at.sharedSizeBytes));
  if (kPreferShared) HXM_CUDA_TRY(cudaFuncSetAttribute(Kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  done.fetch_or(bit, std::memory_order_release);
  return HXM_OK;
}

}  // namespace hxm
