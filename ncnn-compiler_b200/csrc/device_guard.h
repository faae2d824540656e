// The CUDA device of a call.
#pragma once

#include <cuda_runtime.h>

namespace nb {

// Makes the model's device current for the duration of a call and puts the caller's device back:
// a process may hold one handle per GPU and call them in any order from one thread.
struct DeviceGuard {
  int previous = -1;
  bool switched = false;
  explicit DeviceGuard(int device) {
    if (device < 0) return;
    if (cudaGetDevice(&previous) != cudaSuccess) {
      previous = -1;
      cudaGetLastError();
    }
    if (previous != device) switched = cudaSetDevice(device) == cudaSuccess && previous >= 0;
  }
  ~DeviceGuard() {
    if (switched) cudaSetDevice(previous);
  }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
};

}  // namespace nb
