// What every extern "C" entry of libmuspace_ops.so shares: a status code and a
// per-thread message in place of exceptions, and the current device restored.
#pragma once

#include <cuda_runtime.h>

#include <string>

#include "../../include/muspace_msda.h"

namespace capi {

extern thread_local std::string g_last_error;

struct Failure {
  int status;
};

[[noreturn]] inline void fail(int status, const std::string& msg) {
  g_last_error = msg;
  throw Failure{status};
}

inline void require(bool ok, const std::string& msg) {
  if (!ok) fail(MSDA_STATUS_INVALID_ARGUMENT, msg);
}

inline void check_launch(cudaError_t err, const char* what) {
  if (err != cudaSuccess)
    fail(MSDA_STATUS_CUDA_ERROR, std::string(what) + ": " + cudaGetErrorName(err) + ": " + cudaGetErrorString(err));
}

// Makes `device` current for the launch and restores the caller's device.
struct DeviceGuard {
  int previous = -1;
  explicit DeviceGuard(int device) {
    if (cudaGetDevice(&previous) != cudaSuccess) previous = -1;
    if (previous != device) check_launch(cudaSetDevice(device), "cudaSetDevice");
  }
  ~DeviceGuard() {
    int now = -1;
    if (previous >= 0 && cudaGetDevice(&now) == cudaSuccess && now != previous) cudaSetDevice(previous);
  }
};

template <typename F>
int guarded(F&& body) {
  try {
    body();
    g_last_error.clear();
    return MSDA_STATUS_OK;
  } catch (const Failure& f) {
    return f.status;
  } catch (...) {
    g_last_error = "internal error";
    return MSDA_STATUS_CUDA_ERROR;
  }
}

}  // namespace capi
