// norm_rows.cu -- row operators around the RACE layer: the residual addition with
// its root-mean-square norm (forward, backward, and with 8-bit output rows), the
// SwiGLU product as 8-bit rows, and the conversion of rows to and from 8 bits.
//
// Mathematics, one row of K values at a time:
//   h = round_T(x + r)            (the residual stream is held in the tensors' type T)
//   rstd = 1 / sqrt(mean(h^2) + eps),   y = h * rstd * w
//   backward, g = dy * w:  dx = dr = rstd * (g - h * rstd^2 * mean(g * h)) + dh,
//                          dw = sum over rows of dy * h * rstd
//   8-bit row of y: scale = max|y| / 127, q = round_to_even(y / scale)
// Sums, statistics and everything up to the last rounding are fp32.
//
// A row of zeros has scale 0 and q = 0.  A row that holds a NaN (or whose largest
// magnitude is infinite) has scale NaN (infinity), so whatever is computed from it
// is not finite either; no such row touches another.
#include "race_b200.h"

#include <math.h>
#include <stdio.h>

#include "common.cuh"
#include "internal.h"

namespace {

using race::err;
using race::from_f;
using race::launched;
using race::to_f;

constexpr int kNT = 256;  // threads of a block that owns one row

enum Mode { kNorm = 0, kNormInt8 = 1, kSwigluInt8 = 2, kQuantInt8 = 3 };

struct RowArgs {
  const void *x, *r, *w;
  void *y, *h;
  int8_t *q;
  float *scale, *rstd;
  long long rows, x_stride, r_stride, q_stride;
  int K, w_bf16;
  float eps;
};

__device__ __forceinline__ float weight_at(const void *w, int w_bf16, long long i) {
  if (!w) return 1.f;
  return w_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(w)[i]) : static_cast<const float *>(w)[i];
}

// Sum / largest |value| over the block, the same in every thread and run.
__device__ __forceinline__ float block_sum(float v, float *red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t += red[i];
  return t;
}
// The largest of the bit patterns of |v|: for non-negative floats the order of the
// patterns is the order of the values, with NaN above infinity, so a NaN is kept.
__device__ __forceinline__ uint32_t block_max_bits(uint32_t v, float *red) {
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = __uint_as_float(v);
  __syncthreads();
  uint32_t t = 0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t = max(t, __float_as_uint(red[i]));
  return t;
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// q = round(y / scale).  The product with 127 / amax stands for the division except
// where that factor would overflow (rows of magnitudes near the smallest floats).
struct Quantiser {
  float scale, inv;
  bool tiny;
  __device__ __forceinline__ explicit Quantiser(uint32_t amax_bits) {
    const float amax = __uint_as_float(amax_bits);
    scale = amax / 127.f;
    tiny = amax < 1e-30f;
    inv = tiny ? 0.f : 127.f / amax;
  }
  __device__ __forceinline__ int operator()(float y) const {
    if (tiny) return scale > 0.f ? __float2int_rn(y / scale) : 0;
    return __float2int_rn(y * inv);
  }
};

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.f + __expf(-g)) * u; }

// Any width: the row is read again for each of its passes (from the caches).
template <typename T, int MODE>
__global__ void __launch_bounds__(kNT) row_loop_kernel(RowArgs a) {
  __shared__ float red[32];
  const long long row = blockIdx.x;
  const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
  const T *r = a.r ? static_cast<const T *>(a.r) + row * a.r_stride : nullptr;
  T *h = static_cast<T *>(a.h) + row * a.K;
  const int K = a.K;
  float rstd = 1.f;
  auto stream = [&](int i) {  // h
    float v = to_f<T>(x[i]);
    if (r) v = to_f<T>(from_f<T>(v + to_f<T>(r[i])));
    return v;
  };
  if (MODE == kNorm || MODE == kNormInt8) {
    float ss = 0.f;
    for (int i = threadIdx.x; i < K; i += kNT) {
      const float v = stream(i);
      ss = fmaf(v, v, ss);
    }
    rstd = rsqrtf(block_sum(ss, red) / (float)K + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
  }
  auto value = [&](int i) {
    if (MODE == kSwigluInt8) return silu_mul(to_f<T>(x[i]), to_f<T>(x[(long long)K + i]));
    if (MODE == kQuantInt8) return to_f<T>(x[i]);
    return stream(i) * rstd * weight_at(a.w, a.w_bf16, i);
  };
  if (MODE == kNorm) {
    T *y = static_cast<T *>(a.y) + row * K;
    for (int i = threadIdx.x; i < K; i += kNT) {
      const float v = stream(i);
      y[i] = from_f<T>(v * rstd * weight_at(a.w, a.w_bf16, i));
      if (r) h[i] = from_f<T>(v);
    }
    return;
  }
  uint32_t m = 0;
  for (int i = threadIdx.x; i < K; i += kNT) m = max(m, abs_bits(value(i)));
  const Quantiser qz(block_max_bits(m, red));
  if (threadIdx.x == 0) a.scale[row] = qz.scale;
  int8_t *q = a.q + row * a.q_stride;
  for (int i = threadIdx.x; i < K; i += kNT) {
    q[i] = (int8_t)qz(value(i));
    if (MODE == kNormInt8 && r) h[i] = from_f<T>(stream(i));
  }
}

struct BwdArgs {
  const void *dy, *dh, *h, *w;
  const float *rstd;
  void *dx, *dw;
  float *part;  // [blocks, K] partial sums of dw
  long long rows;
  int K, w_bf16;
};

// Any width: a block takes rows blockIdx.x, blockIdx.x + gridDim.x, ...; its share of
// dw is kept in its own row of `part`, in a fixed order.
template <typename T>
__global__ void __launch_bounds__(kNT) bwd_loop_kernel(BwdArgs a) {
  __shared__ float red[32];
  const int K = a.K;
  float *part = a.part ? a.part + (long long)blockIdx.x * K : nullptr;
  if (part)
    for (int i = threadIdx.x; i < K; i += kNT) part[i] = 0.f;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *dy = static_cast<const T *>(a.dy) + row * K;
    const T *dh = a.dh ? static_cast<const T *>(a.dh) + row * K : nullptr;
    const T *h = static_cast<const T *>(a.h) + row * K;
    T *dx = static_cast<T *>(a.dx) + row * K;
    const float rstd = a.rstd[row];
    float s = 0.f;
    for (int i = threadIdx.x; i < K; i += kNT)
      s = fmaf(to_f<T>(dy[i]) * weight_at(a.w, a.w_bf16, i), to_f<T>(h[i]) * rstd, s);
    const float c = block_sum(s, red) / (float)K;
    for (int i = threadIdx.x; i < K; i += kNT) {
      const float d = to_f<T>(dy[i]), xh = to_f<T>(h[i]) * rstd;
      float v = rstd * (d * weight_at(a.w, a.w_bf16, i) - xh * c);
      if (dh) v += to_f<T>(dh[i]);
      dx[i] = from_f<T>(v);
      if (part) part[i] = fmaf(d, xh, part[i]);
    }
  }
}

// dw[k] = sum of the blocks' partial sums, in their order.
__global__ void __launch_bounds__(256) dw_sum_kernel(const float *part, int n, int K, void *dw, int w_bf16) {
  __shared__ float red[8][32];
  const int k = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
  float s = 0.f;
  if (k < K)
    for (int i = g; i < n; i += 8) s += part[(long long)i * K + k];
  red[g][threadIdx.x & 31] = s;
  __syncthreads();
  if (g == 0 && k < K) {
    s = 0.f;
    for (int i = 0; i < 8; ++i) s += red[i][threadIdx.x];
    if (w_bf16)
      static_cast<__nv_bfloat16 *>(dw)[k] = __float2bfloat16_rn(s);
    else
      static_cast<float *>(dw)[k] = s;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) dequant_kernel(const int8_t *q, long long q_stride, const float *scale, T *out,
                                                      long long rows, int K) {
  const long long row = blockIdx.x;
  const float s = scale[row];
  for (int i = blockIdx.y * 256 + threadIdx.x; i < K; i += gridDim.y * 256)
    out[row * K + i] = from_f<T>((float)q[row * q_stride + i] * s);
}

// ------------------------------------------------------------------ host side
int check_rows(const char *what, int64_t rows, int64_t K, int dtype) {
  char buf[160];
  if (dtype != RACE_F32 && dtype != RACE_BF16) {
    snprintf(buf, sizeof(buf), "%s: dtype %d", what, dtype);
    return race::report_error(RACE_ERR_DTYPE, buf);
  }
  // the grid has a block per row; a row index times a row's length is 64-bit
  if (rows < 1 || rows > 0x7fffffffLL || K < 1 || K > (1 << 24)) {
    snprintf(buf, sizeof(buf), "%s: rows=%lld (1..2^31-1), width=%lld (1..2^24)", what, (long long)rows, (long long)K);
    return race::report_error(RACE_ERR_SHAPE, buf);
  }
  return RACE_OK;
}

template <int MODE>
int launch_rows(const char *what, const RowArgs &a, int dtype, cudaStream_t s) {
  if (dtype == RACE_BF16)
    row_loop_kernel<__nv_bfloat16, MODE><<<(unsigned)a.rows, kNT, 0, s>>>(a);
  else
    row_loop_kernel<float, MODE><<<(unsigned)a.rows, kNT, 0, s>>>(a);
  return launched(what);
}

// blocks of the backward: each keeps one row of partial sums of dw
int bwd_blocks(int64_t rows) { return (int)(rows < 1184 ? rows : 1184); }

}  // namespace

extern "C" {

int race_rms_norm_fwd(const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, int dtype,
                      const void *weight, int weight_dtype, void *y, void *h, float *rstd, int64_t rows, int64_t K,
                      float eps, void *stream) {
  if (!x || !y || (residual && !h)) return err(RACE_ERR_ARG, "race_rms_norm_fwd: null pointer");
  if (const int rc = check_rows("race_rms_norm_fwd", rows, K, dtype)) return rc;
  if (weight && weight_dtype != RACE_F32 && weight_dtype != RACE_BF16)
    return err(RACE_ERR_DTYPE, "race_rms_norm_fwd: weight dtype %lld", weight_dtype);
  if (x_stride < K || (residual && residual_stride < K)) return err(RACE_ERR_SHAPE, "race_rms_norm_fwd: row stride below the width %lld", K);
  RowArgs a{x, residual, weight, y, h, nullptr, nullptr, rstd, rows, x_stride, residual_stride, 0, (int)K, weight_dtype == RACE_BF16, eps};
  return launch_rows<kNorm>("rms_norm_fwd", a, dtype, reinterpret_cast<cudaStream_t>(stream));
}

int race_rms_norm_int8(const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, int dtype,
                       const void *weight, int weight_dtype, int8_t *q, int64_t q_stride, float *scale, void *h,
                       int64_t rows, int64_t K, float eps, void *stream) {
  if (!x || !q || !scale || (residual && !h)) return err(RACE_ERR_ARG, "race_rms_norm_int8: null pointer");
  if (const int rc = check_rows("race_rms_norm_int8", rows, K, dtype)) return rc;
  if (weight && weight_dtype != RACE_F32 && weight_dtype != RACE_BF16)
    return err(RACE_ERR_DTYPE, "race_rms_norm_int8: weight dtype %lld", weight_dtype);
  if (x_stride < K || q_stride < K || (residual && residual_stride < K))
    return err(RACE_ERR_SHAPE, "race_rms_norm_int8: row stride below the width %lld", K);
  RowArgs a{x, residual, weight, nullptr, h, q, scale, nullptr, rows, x_stride, residual_stride, q_stride, (int)K, weight_dtype == RACE_BF16, eps};
  return launch_rows<kNormInt8>("rms_norm_int8", a, dtype, reinterpret_cast<cudaStream_t>(stream));
}

int race_quant_int8(const void *x, int64_t x_stride, int dtype, int8_t *q, int64_t q_stride, float *scale, int64_t rows,
                    int64_t K, void *stream) {
  if (!x || !q || !scale) return err(RACE_ERR_ARG, "race_quant_int8: null pointer");
  if (const int rc = check_rows("race_quant_int8", rows, K, dtype)) return rc;
  if (x_stride < K || q_stride < K) return err(RACE_ERR_SHAPE, "race_quant_int8: row stride below the width %lld", K);
  RowArgs a{x, nullptr, nullptr, nullptr, nullptr, q, scale, nullptr, rows, x_stride, 0, q_stride, (int)K, 0, 0.f};
  return launch_rows<kQuantInt8>("quant_int8", a, dtype, reinterpret_cast<cudaStream_t>(stream));
}

int race_swiglu_int8(const void *gate_up, int64_t stride, int dtype, int8_t *q, int64_t q_stride, float *scale,
                     int64_t rows, int64_t F, void *stream) {
  if (!gate_up || !q || !scale) return err(RACE_ERR_ARG, "race_swiglu_int8: null pointer");
  if (const int rc = check_rows("race_swiglu_int8", rows, F, dtype)) return rc;
  if (stride < 2 * F || q_stride < F) return err(RACE_ERR_SHAPE, "race_swiglu_int8: row stride below the width (F=%lld)", F);
  RowArgs a{gate_up, nullptr, nullptr, nullptr, nullptr, q, scale, nullptr, rows, stride, 0, q_stride, (int)F, 0, 0.f};
  return launch_rows<kSwigluInt8>("swiglu_int8", a, dtype, reinterpret_cast<cudaStream_t>(stream));
}

int race_dequant_int8(const int8_t *q, int64_t q_stride, const float *scale, void *out, int dtype, int64_t rows,
                      int64_t K, void *stream) {
  if (!q || !scale || !out) return err(RACE_ERR_ARG, "race_dequant_int8: null pointer");
  if (const int rc = check_rows("race_dequant_int8", rows, K, dtype)) return rc;
  if (q_stride < K) return err(RACE_ERR_SHAPE, "race_dequant_int8: row stride below the width %lld", K);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)rows, (unsigned)((K + 1023) / 1024 < 64 ? (K + 1023) / 1024 : 64));
  if (dtype == RACE_BF16)
    dequant_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(q, q_stride, scale, static_cast<__nv_bfloat16 *>(out), rows, (int)K);
  else
    dequant_kernel<float><<<grid, 256, 0, s>>>(q, q_stride, scale, static_cast<float *>(out), rows, (int)K);
  return launched("dequant_int8");
}

size_t race_rms_norm_bwd_workspace_bytes(int64_t rows, int64_t K) {
  if (rows < 1 || K < 1) return 0;
  return sizeof(float) * (size_t)bwd_blocks(rows) * (size_t)K;
}

int race_rms_norm_bwd(const void *dy, const void *dh, const void *h, const float *rstd, int dtype, const void *weight,
                      int weight_dtype, void *dx, void *dw, int64_t rows, int64_t K, void *workspace,
                      size_t workspace_bytes, void *stream) {
  if (!dy || !h || !rstd || !dx) return err(RACE_ERR_ARG, "race_rms_norm_bwd: null pointer");
  if (const int rc = check_rows("race_rms_norm_bwd", rows, K, dtype)) return rc;
  if ((weight || dw) && weight_dtype != RACE_F32 && weight_dtype != RACE_BF16)
    return err(RACE_ERR_DTYPE, "race_rms_norm_bwd: weight dtype %lld", weight_dtype);
  if (dw && (!workspace || workspace_bytes < race_rms_norm_bwd_workspace_bytes(rows, K)))
    return err(RACE_ERR_WORKSPACE, "race_rms_norm_bwd: workspace of %lld bytes needed", (long long)race_rms_norm_bwd_workspace_bytes(rows, K));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int blocks = bwd_blocks(rows);
  BwdArgs a{dy, dh, h, weight, rstd, dx, dw, dw ? static_cast<float *>(workspace) : nullptr, rows, (int)K, weight_dtype == RACE_BF16};
  if (dtype == RACE_BF16)
    bwd_loop_kernel<__nv_bfloat16><<<blocks, kNT, 0, s>>>(a);
  else
    bwd_loop_kernel<float><<<blocks, kNT, 0, s>>>(a);
  if (const int rc = launched("rms_norm_bwd")) return rc;
  if (!dw) return RACE_OK;
  dw_sum_kernel<<<(unsigned)((K + 31) / 32), 256, 0, s>>>(a.part, blocks, (int)K, dw, weight_dtype == RACE_BF16);
  return launched("rms_norm_bwd dw");
}

}  // extern "C"
