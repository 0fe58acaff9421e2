#pragma once
// Host services of gemm.cu that the library's other translation units use.
#include <cuda.h>

#include <cstddef>
#include <cstdint>

namespace mxfp6 {
namespace host {

// Error state of this thread (mxfp6_last_error): clear() at the start of a call, fail() prints
// "[mxfp6] <message>", records the code and returns it.
void clear();
int fail(int code, const char* message);

int device();     // current device, or -1
int sm_count();   // of the current device; 148 without one
long long wait_budget();  // cycles a kernel's bounded waits may take (mxfp6_set_wait_budget)

// Packed FP6 matrix read in 128 (K) x box_rows boxes through the 16U6 unpack mode; false on failure.
bool fp6_tmap(CUtensorMap* map, const void* ptr, int rows, int Kp, int row_bytes, int box_rows);
// Byte matrix [rows][row_bytes] read in 128-byte x box_rows boxes with 128-byte swizzle.
bool bytes_tmap(CUtensorMap* map, const void* ptr, int rows, int row_bytes, int box_rows);

}  // namespace host

// Status bits of moe.cu's kernels: read and cleared by mxfp6_device_status(). False when a copy failed.
bool take_moe_status(unsigned int* bits);

}  // namespace mxfp6
