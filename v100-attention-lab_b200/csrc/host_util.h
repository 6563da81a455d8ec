// Host-side helpers shared by the entry points of the recurrent and windowed
// operators: the device check and the error of a failed runtime call.
#pragma once
#include <cuda_runtime.h>

#include "../../include/gdn_b200.h"

namespace gdn {

constexpr int kMaxDevices = 64;

// Whether the current device is an sm_100 one; its index in *dev.
inline bool device_is_sm100(int* dev_out) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
    cudaGetLastError();
    return false;
  }
  static int cached[kMaxDevices] = {0};  // 0 unknown, 1 yes, 2 no
  if (cached[dev] == 0) {
    int major = 0, minor = 0;
    cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
    cached[dev] = (major == 10 && minor == 0) ? 1 : 2;
  }
  *dev_out = dev;
  return cached[dev] == 1;
}

// Status of a failed runtime call; leaves no error behind for the caller's own
// checks.
inline int cuda_failed() {
  cudaGetLastError();
  return GDN_ERR_CUDA;
}

inline int dtype_size(int dt) { return dt == GDN_DTYPE_F32 ? 4 : 2; }

}  // namespace gdn
