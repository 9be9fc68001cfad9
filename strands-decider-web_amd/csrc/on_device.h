// The calling thread's current device is the caller's again after a call.
#pragma once
#include <hip/hip_runtime.h>

namespace ha {

struct OnDevice {
  int before = -1;
  hipError_t rc;
  explicit OnDevice(int device) {
    rc = hipGetDevice(&before);
    if (rc == hipSuccess && before != device) rc = hipSetDevice(device);
    else before = -1;
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

}  // namespace ha
