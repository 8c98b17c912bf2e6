// device_scope.hpp -- the calls that run between a program's own work on the
// GPU make the context's device current and set the program's back.
#pragma once

#include <hip/hip_runtime_api.h>

namespace vsk {

class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (hipGetDevice(&before_) != hipSuccess) before_ = device;
    other_ = before_ != device;
    if (other_) (void)hipSetDevice(device);
  }
  ~DeviceScope() {
    if (other_) (void)hipSetDevice(before_);
  }
  DeviceScope(const DeviceScope &) = delete;
  DeviceScope &operator=(const DeviceScope &) = delete;

 private:
  int before_ = 0;
  bool other_ = false;
};

}  // namespace vsk
