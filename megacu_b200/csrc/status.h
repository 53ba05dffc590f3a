// Status values and the device guard shared by the routing and 4-bit entry
// points.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include <megacu_b200.h>

namespace megacu_b200 {

inline megacu_status ok_status() { return {MEGACU_OK, 0, nullptr}; }

inline megacu_status fail(megacu_status_code code, std::uint16_t detail, char const *msg) {
  return {static_cast<std::uint8_t>(code), detail, msg};
}

inline megacu_status cuda_fail(cudaError_t e, std::uint16_t detail) {
  return {MEGACU_LAUNCH_ERROR, detail, cudaGetErrorString(e)};
}

inline bool aligned_to(void const *p, std::uintptr_t bytes) {
  return (reinterpret_cast<std::uintptr_t>(p) & (bytes - 1)) == 0;
}

// Makes `device` current for the launches of one call and the caller's device
// current again after it.
class device_guard {
 public:
  explicit device_guard(int device) {
    status_ = cudaGetDevice(&before_);
    if (status_ == cudaSuccess && before_ != device) {
      status_ = cudaSetDevice(device);
      restore_ = status_ == cudaSuccess;
    }
  }
  ~device_guard() {
    if (restore_) cudaSetDevice(before_);
  }
  device_guard(device_guard const &) = delete;
  device_guard &operator=(device_guard const &) = delete;
  cudaError_t status() const { return status_; }

 private:
  cudaError_t status_ = cudaSuccess;
  int before_ = 0;
  bool restore_ = false;
};

}  // namespace megacu_b200
