// Status codes and messages of the C entry points, shared by the library's
// translation units.
#pragma once

#include <string>

#include "common.cuh"

namespace scmp {

inline thread_local std::string t_last_error;

inline int fail(int code, const std::string& msg) {
  t_last_error = msg;
  return code;
}
inline int cuda_fail(cudaError_t e, const char* what) {
  return fail(SCMP_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}
#define SCMP_CUDA(call, what)                  \
  do {                                         \
    cudaError_t e_ = (call);                   \
    if (e_ != cudaSuccess) return cuda_fail(e_, what); \
  } while (0)

// The device error record of the linear layer's translation unit, read and cleared
// (the device is synchronised by the caller).
cudaError_t linears_device_error(DeviceError* out);

}  // namespace scmp
