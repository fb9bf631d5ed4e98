// internal.h -- helpers shared between the library's translation units
// (defined in race_api.cu; not part of the C ABI).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "race_b200.h"

namespace race {
int report_error(int code, const char *msg);  // sets race_last_error(), returns code
void clear_error();
void note_launch();  // bumps race_launch_counter()

uint32_t current_wait_limit();  // race_set_wait_limit()'s value for the next launch
bool status_check_on();         // race_set_status_check()
bool withhold_first_load();     // race_test_withhold_first_load()
// Tensor map of rows x cols bytes (row stride a multiple of 16 bytes) in boxes of
// box_rows x 128 bytes, 128-byte swizzle; out-of-range bytes read as 0.  False if the
// driver refuses it.  `map` points at a CUtensorMap.
bool make_byte_rows_map(void *map, const void *base, int64_t rows, int64_t cols, int64_t row_stride, int box_rows);

uint32_t current_wait_limit();  // race_set_wait_limit()'s value for the next launch
bool status_check_on();         // race_set_status_check()
bool withhold_first_load();     // race_test_withhold_first_load()
// Tensor map of rows x cols bytes (row stride a multiple of 16 bytes) in boxes of
// box_rows x 128 bytes, 128-byte swizzle; out-of-range bytes read as 0.  False if the
// driver refuses it.  `map` points at a CUtensorMap.
bool make_byte_rows_map(void *map, const void *base, int64_t rows, int64_t cols, int64_t row_stride, int box_rows);

// Fails with `code`: formats the detail of race_last_error().
inline int err(int code, const char *fmt, long long a = 0, long long b = 0) {
  char buf[256];
  snprintf(buf, sizeof(buf), fmt, a, b);
  return report_error(code, buf);
}
inline int cuda_err(const char *what, cudaError_t e) {
  char buf[256];
  snprintf(buf, sizeof(buf), "%s: %s", what, cudaGetErrorString(e));
  return report_error(RACE_ERR_CUDA, buf);
}
// After a launch: counts it, and turns its error into a status.
inline int launched(const char *what) {
  note_launch();
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_err(what, e);
  clear_error();
  return RACE_OK;
}
}  // namespace race
