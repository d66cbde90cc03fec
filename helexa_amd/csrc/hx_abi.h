// What the files of the C ABI share: statuses with a message, the current device.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hx_moe.h"

namespace hx {

// sets hx_last_error()'s text on this thread and returns code
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

#define HX_HIP(call)                                                                               \
  do {                                                                                             \
    hipError_t e_ = (call);                                                                        \
    if (e_ != hipSuccess) return fail(HX_ERR_DEVICE, "%s failed: %s (%s:%d)", #call, hipGetErrorString(e_), \
                                      __FILE__, __LINE__);                                         \
  } while (0)

inline bool capturing(hipStream_t s) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  (void)hipStreamIsCapturing(s, &st);
  return st != hipStreamCaptureStatusNone;
}

// whether the n bytes at a and the m bytes at b have one in common
inline bool overlap(const void* a, size_t n, const void* b, size_t m) {
  return (uintptr_t)a < (uintptr_t)b + m && (uintptr_t)b < (uintptr_t)a + n;
}

// a handle's device as the current one, and the caller's again
struct DeviceScope {
  int was = -1;
  hipError_t err;
  explicit DeviceScope(int device) {
    if ((err = hipGetDevice(&was)) != hipSuccess) return;
    if (was == device) was = -1;
    else err = hipSetDevice(device);
  }
  ~DeviceScope() {
    if (was >= 0) (void)hipSetDevice(was);
  }
};

// token counts above this are refused by every entry point: the kernels index
// the T * k assignments with 32-bit integers (k <= HX_MAX_TOPK)
constexpr int64_t HX_MAX_TOKENS = (int64_t)1 << 24;

}  // namespace hx
