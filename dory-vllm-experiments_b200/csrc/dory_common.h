// dory_common.h — what the library's translation units share on the host side: the calling
// thread's last error (dory_decode_last_error) and small argument helpers.
#ifndef DORY_COMMON_H_
#define DORY_COMMON_H_

#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/dory_decode.h"

namespace dory {

// Records `message` as the calling thread's last error and returns `status`.
__attribute__((visibility("hidden"))) int32_t set_error(int32_t status, const char* message);

__attribute__((format(printf, 2, 3))) inline int32_t fail(int32_t status, const char* fmt, ...) {
  char text[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  return set_error(status, text);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// SMs of the current device, whose number goes to *device; 0 on failure.
inline int device_sms(int* device) {
  static int counts[64] = {0};
  if (cudaGetDevice(device) != cudaSuccess || *device < 0 || *device >= 64) return 0;
  if (!counts[*device]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *device) == cudaSuccess)
      counts[*device] = n;
  }
  return counts[*device];
}

// The status of a kernel launch just made.
inline int32_t launched(cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return fail(DORY_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  return DORY_OK;
}

}  // namespace dory

#endif  // DORY_COMMON_H_
