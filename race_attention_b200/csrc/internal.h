// internal.h -- helpers shared between the library's translation units
// (defined in race_api.cu; not part of the C ABI).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <initializer_list>

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
// driver refuses it.  `map` points at a CUtensorMap.  A thread that has only queried the
// runtime calls bind_context() first.
bool bind_context();
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
// RACE_ERR_ALIGN where an array does not start at a multiple of its values' size (no access of a
// kernel to it would be aligned); absent arrays are NULL.
struct Values {
  const void *at;
  int size;  // of a value, in bytes
};
inline int check_values(const char *what, std::initializer_list<Values> arrays) {
  char buf[160];
  for (const Values &v : arrays)
    if (reinterpret_cast<uintptr_t>(v.at) % (uintptr_t)v.size) {
      snprintf(buf, sizeof(buf), "%s: a tensor does not start at a multiple of its values' size", what);
      return report_error(RACE_ERR_ALIGN, buf);
    }
  return RACE_OK;
}
inline int value_size(int dtype) { return dtype == RACE_F32 ? 4 : 2; }
// Launch of a kernel that starts with wait_for_predecessor(): with the stream's previous kernel
// still running (once all of its blocks are past let_successor_start(), or done), so that its
// launch and whatever it does before that call overlap it.
template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, unsigned cluster,
                         const A &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
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
