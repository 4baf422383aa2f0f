// What the kernels of the paged key-value cache share: status records, the device of a call, and the checks of
// addresses and strides.
#pragma once
#include <limits.h>

#include <initializer_list>

#include "host_util.h"
#include "ptx.cuh"

namespace syn {

// Keeps the first record; the launch carries on without the offending access.
__device__ __forceinline__ void paged_record(int32_t* status, int code, int who, int value) {
  if (status != nullptr && atomicCAS(status, 0, code) == 0) {
    status[1] = who;
    status[2] = value;
    status[3] = static_cast<int>(blockIdx.x);
  }
}

// Makes the device that owns a call's tensors the current one for the launch.
class PagedDevice {
 public:
  explicit PagedDevice(int device) {
    if (device < 0) return;
    err_ = cudaGetDevice(&before_);
    if (err_ == cudaSuccess && before_ != device) {
      err_ = cudaSetDevice(device);
      changed_ = err_ == cudaSuccess;
    }
  }
  ~PagedDevice() {
    if (changed_) cudaSetDevice(before_);
  }
  PagedDevice(const PagedDevice&) = delete;
  PagedDevice& operator=(const PagedDevice&) = delete;
  cudaError_t error() const { return err_; }

 private:
  int before_ = 0;
  bool changed_ = false;
  cudaError_t err_ = cudaSuccess;
};

inline bool paged_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Strides of a tensor with `extent[i]` entries along axis i and elements of `size` bytes: positive and
// multiples of 16 bytes, but for an axis of one entry, whose stride says nothing and becomes 0.
inline bool paged_strides(int64_t* s, std::initializer_list<int> extent, int size) {
  for (int n : extent) {
    if (n <= 1) *s = 0;
    else if (*s <= 0 || ((*s * size) & 15) != 0) return false;
    ++s;
  }
  return true;
}

}  // namespace syn
