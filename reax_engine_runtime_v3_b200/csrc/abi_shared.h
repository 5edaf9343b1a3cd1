// Host helpers of the C ABI that its translation units share (defined in abi.cu).
#pragma once

#include <cuda_runtime.h>

namespace reax_abi {

// Record a message for reax_last_error() on this thread and return `code`.
int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);

// Multiprocessors of the current device, which must be an sm_100 GPU.
int current_sms(int* sms);
// Multiprocessors of `device` (-1: the current one); -1 on failure.
int device_sms(int device);

// Bound of device-side waits (reax_set_wait_timeout_ns).
unsigned long long wait_timeout_ns();

}  // namespace reax_abi
