// Host helpers of the C ABI that its translation units share (defined in abi.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

namespace reax_abi {

// Record a message for reax_last_error() on this thread and return `code`.
int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);

// Multiprocessors of the current device, which must be an sm_100 GPU.
int current_sms(int* sms);
// Multiprocessors of `device` (-1: the current one); -1 on failure.
int device_sms(int device);

// Tensor map of row-major bf16 [rows, cols], row stride ld elements; boxes of box_rows x box_cols, zeros outside.
int encode_rows(CUtensorMap* map, const void* base, int cols, int rows, long long ld, int box_cols, int box_rows);
// Tensor map of contiguous rows of `dim` (64, 128 or 256) 8-bit codes; boxes of min(dim, 128) codes by box_rows rows, 128-byte
// swizzle (64-byte where dim is 64).
int encode_codes(CUtensorMap* map, const void* base, int dim, long long rows, int box_rows);
// Bound of device-side waits (reax_set_wait_timeout_ns).
unsigned long long wait_timeout_ns();

}  // namespace reax_abi
