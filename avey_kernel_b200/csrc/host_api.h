// Host-side services that the translation units of the library share: one
// last-error string per thread, one launch counter, the device checks and the
// tensor-map encoder (all defined in avey_api.cu).
#pragma once

#include <cuda.h>
#include <cstdint>

namespace avey_host {

int set_error(int code, const char* msg);
int clear_error();
void count_launches(int n);

// AVEY_OK when the current device is sm_100, else the error it recorded.
int device_ok();

// Multiprocessors of the current device.
int multiprocessors();

// Encode a 3-D tiled map of 16-bit elements (dtype AVEY_BF16 / AVEY_F16): dims
// {inner, rows, batch}, strides in bytes, a box of 64 inner elements (128-byte
// swizzle) by box_rows rows, zero fill out of bounds.
int encode_rows16(int dtype, const void* base, uint64_t inner, uint64_t rows, uint64_t batch, uint64_t row_bytes,
                  uint64_t batch_bytes, int box_rows, CUtensorMap* map);

// The same for output tiles of 32 rows of 64 bytes (64-byte swizzle): 32 16-bit
// or, with dtype AVEY_F32, 16 32-bit elements.
int encode_tiles(int dtype, void* base, uint64_t inner, uint64_t rows, uint64_t batch, uint64_t row_bytes,
                 uint64_t batch_bytes, CUtensorMap* map);

// Test hook (avey_test_hooks_v1): launches are to stall.
bool test_stall();

// The status word (read, and reset with `clear`) and the wait limit of the
// kernels of avey_linear.cu, on the current device; a cudaError_t.
int linear_flags(unsigned int* flags, bool clear);
int linear_wait_limit(long long cycles);

}  // namespace avey_host
