// Runs an entry point's body with the device of its stream current (the default stream is the current device's), so that
// launches land where the tensors are, and turns what escapes into a status.
#pragma once

#include <hip/hip_runtime.h>

#include <exception>

#include "host_support.hpp"
#include "launch.hpp"

namespace tcu {

template <typename Body>
inline int on_stream_device(const char *what, void *stream, Body &&body) {
  try {
    const unsigned long before = launch_count();
    int current = 0;
    bool moved = false;
    if (stream) {
      hipDevice_t of_stream = 0;
      hipError_t e = hipStreamGetDevice(static_cast<hipStream_t>(stream), &of_stream);
      if (e == hipSuccess) e = hipGetDevice(&current);
      if (e == hipSuccess && (int)of_stream != current) {
        e = hipSetDevice((int)of_stream);
        moved = e == hipSuccess;
      }
      if (e != hipSuccess) {
        (void)hipGetLastError();
        return report_failure(TCU_ERR_RUNTIME, std::string(what) + ": device of the stream: " + hipGetErrorString(e));
      }
    }
    const int rc = launch_outcome(what, before, body());
    if (moved) (void)hipSetDevice(current);
    return rc;
  } catch (const std::exception &) {  // out of host memory; no message, which would need some
    return TCU_ERR_RUNTIME;
  }
}

}  // namespace tcu
