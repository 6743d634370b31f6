// Runs an entry point's body with the device of its stream current (the default stream is the current device's), so that
// launches land where the tensors are, and turns what escapes into a status.
#pragma once

#include <hip/hip_runtime.h>

#include "host_support.hpp"
#include "launch.hpp"

namespace tcu {

// makes `device` current again when it goes out of scope
struct DeviceBack {
  int device = -1;
  ~DeviceBack() {
    if (device >= 0) (void)hipSetDevice(device);
  }
};

template <typename Body>
inline int on_stream_device(const char *what, void *stream, Body &&body) {
  try {
    DeviceBack back;
    const unsigned long before = launch_count();
    if (stream) {
      int current = 0;
      hipDevice_t of_stream = 0;
      hipError_t e = hipStreamGetDevice(static_cast<hipStream_t>(stream), &of_stream);
      if (e == hipSuccess) e = hipGetDevice(&current);
      if (e == hipSuccess && (int)of_stream != current) {
        e = hipSetDevice((int)of_stream);
        if (e == hipSuccess) back.device = current;
      }
      if (e != hipSuccess) {
        (void)hipGetLastError();
        return report_failure(TCU_ERR_RUNTIME, std::string(what) + ": device of the stream: " + hipGetErrorString(e));
      }
    }
    return launch_outcome(what, before, body());
  } catch (...) {  // out of host memory
    try {
      return report_failure(TCU_ERR_RUNTIME, std::string(what) + ": out of host memory");
    } catch (...) {  // not even for the message
      return TCU_ERR_RUNTIME;
    }
  }
}

}  // namespace tcu
