#pragma once

#include <cuda_runtime_api.h>

namespace orion {

// Makes `device` current for the scope and puts the caller's device back afterwards, whatever made another one current meanwhile.
struct ScopedDevice {
  int prev = -1;
  cudaError_t status;
  explicit ScopedDevice(int device) {
    status = cudaGetDevice(&prev);
    if (status == cudaSuccess && prev != device) status = cudaSetDevice(device);
  }
  ~ScopedDevice() {
    int now = -1;
    if (prev >= 0 && cudaGetDevice(&now) == cudaSuccess && now != prev) cudaSetDevice(prev);
  }
};

}  // namespace orion
