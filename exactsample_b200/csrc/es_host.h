// Host-side helpers of the C ABI: the thread's last error, and the checks of
// tensors (dtype, rank, strides, overlap) that its entry points share.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>
#include <numeric>
#include <string>

#include "exactsample_b200.h"

namespace es {
namespace host {
inline thread_local std::string g_error;

inline int fail(int code, const std::string& message) {
  g_error = message;
  return code;
}

inline size_t element_size(int32_t dtype) {
  switch (dtype) {
    case ES_F32: case ES_I32: return 4;
    case ES_F64: case ES_I64: return 8;
    case ES_F16: case ES_BF16: return 2;
    case ES_U8: return 1;
    default: return 0;
  }
}
inline int64_t numel(const es_tensor& t) {
  int64_t n = 1;
  for (int d = 0; d < t.ndim; ++d) n *= t.size[d];
  return n;
}
// [first byte, one past the last byte] of a strided view.
inline bool extent(const es_tensor& t, uintptr_t* begin, uintptr_t* end) {
  if (numel(t) == 0) return false;
  const size_t e = element_size(t.dtype);
  uintptr_t span = e;
  for (int d = 0; d < t.ndim; ++d) span += uintptr_t(t.size[d] - 1) * uintptr_t(t.stride[d]) * e;
  *begin = reinterpret_cast<uintptr_t>(t.data);
  *end = *begin + span;
  return true;
}
// Address intervals prove disjointness (bindings.cpp:25-37).
inline bool disjoint(const es_tensor& a, const es_tensor& b) {
  uintptr_t a0, a1, b0, b1;
  if (!extent(a, &a0, &a1) || !extent(b, &b0, &b1)) return true;
  return a1 <= b0 || b1 <= a0;
}
// A view whose elements never share an address (bindings.cpp:38-44).
inline bool no_internal_overlap(const es_tensor& t) {
  if (numel(t) <= 1) return true;
  for (int d = 0; d < t.ndim; ++d)
    if (t.size[d] > 1 && t.stride[d] == 0) return false;
  if (t.ndim == 1 || t.size[0] <= 1 || t.size[1] <= 1) return true;
  const int64_t divisor = std::gcd(t.stride[0], t.stride[1]);
  return t.size[0] <= t.stride[1] / divisor || t.size[1] <= t.stride[0] / divisor;
}
inline bool check(const es_tensor& t, int32_t dtype, int ndim, const char* name) {
  if (t.dtype != dtype || t.ndim != ndim || (t.data == nullptr && numel(t) != 0)) {
    g_error = std::string(name) + " has wrong device, dtype or rank";
    return false;
  }
  for (int d = 0; d < ndim; ++d)
    if (t.stride[d] < 0 || t.size[d] < 0) {
      g_error = std::string(name) + " has a negative stride";
      return false;
    }
  return true;
}

inline int device_check() {
  static thread_local int checked_device = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(ES_ERR_DEVICE, "no CUDA device is available");
  if (dev == checked_device) return ES_SUCCESS;
  int major = 0;
  if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess || major != 10)
    return fail(ES_ERR_DEVICE, "exactsample_b200 requires an sm_100 (B200) GPU");
  checked_device = dev;
  return ES_SUCCESS;
}
}  // namespace host
}  // namespace es
