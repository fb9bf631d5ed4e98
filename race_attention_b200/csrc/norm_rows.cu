// norm_rows.cu -- row operators around the RACE layer: the residual addition with
// its root-mean-square norm (forward, backward, and with 8-bit output rows), the
// SwiGLU product as 8-bit rows, and the conversion of rows to and from 8 bits.
//
// Mathematics, one row of K values at a time:
//   h = round_T(x + r)            (the residual stream is held in the tensors' type T)
//   rstd = 1 / sqrt(mean(h^2) + eps),   y = h * rstd * w
//   backward, g = dy * w:  dx = dr = rstd * (g - h * rstd^2 * mean(g * h)) + dh,
//                          dw = sum over rows of dy * h * rstd
//   8-bit row of y: scale = max|y| times fp32's 1/127, q = round_to_even(y / scale), the quotient
//                   correctly rounded
// Sums, statistics and everything up to the last rounding are fp32.
//
// A row of zeros (or of values under 2^-143, whose scale fp32 does not hold) has scale 0 and
// q = 0.  A row that holds a NaN (or whose largest magnitude is infinite) has scale NaN
// (infinity), so whatever is computed from it is not finite either; no such row touches another.
#include "race_b200.h"

#include <math.h>
#include <stdio.h>

#include "common.cuh"
#include "internal.h"

namespace {

using race::check_values;
using race::err;
using race::from_f;
using race::launched;
using race::to_f;
using race::value_size;

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
  int q_vec = 0;  // 8-byte stores of 8-bit rows
  float inv_K = 0.f;
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

// four values to signed bytes (the conversion saturates)
__device__ __forceinline__ uint32_t pack_s8(int a, int b, int c, int d) {
  uint32_t r;
  asm("{\n\t.reg .b32 t;\n\t"
      "cvt.pack.sat.s8.s32.b32 t, %4, %3, 0;\n\t"
      "cvt.pack.sat.s8.s32.b32 %0, %2, %1, t;\n\t}"
      : "=r"(r)
      : "r"(a), "r"(b), "r"(c), "r"(d));
  return r;
}

// q = round_to_even(y / scale), where the quotient is rounded to fp32 as a division does: values on
// half a step are common among bf16 rows, and there the last place decides.  Markstein's method: t =
// y (1 / scale), then one step with the residual y - t scale, which the fused multiply-add gives
// exactly; the reciprocal has had a step of Newton's.  On a B200 the result rounds to the same
// integer as the division's for every significand of the scale and every y within four places of
// half a step (all enumerated; of those 3 % are off by the reciprocal alone).  What it costs next to
// that one product: 8-bit norm 32768 x 2048 bf16 72 us and 70.5, rows to 8 bits 37 and 36, 16384 x
// 8192 70 and 64.
// Rows near the ends of fp32's range are first scaled by a power of two (`lift`, which changes no
// quotient), so that their residuals are exact too.  A scale among the subnormals may be well under
// max|y| / 127: such a row's values are held at 127 steps.  Where the scale is 0 or not finite the
// quotients are NaN, and the conversion of a NaN to an integer 0.
struct Quantiser {
  float scale, lift, unit, inv;
  __device__ __forceinline__ explicit Quantiser(uint32_t amax_bits) {
    const float amax = __uint_as_float(amax_bits);
    scale = amax * (1.f / 127.f);
    lift = amax < 1e-25f ? 0x1p100f : amax > 1e30f ? 0x1p-100f : 1.f;
    unit = scale * lift;
    const float y = __fdividef(1.f, unit);
    inv = fmaf(fmaf(-unit, y, 1.f), y, y);
  }
  __device__ __forceinline__ float lifted(float y) const {
    const float most = 127.f * unit;
    return fminf(fmaxf(y * lift, -most), most);
  }
  // quotients (of rows that are lifted: of lifted values)
  template <bool PAIRS>
  __device__ __forceinline__ float2 two(float a, float b) const {
    if constexpr (PAIRS) {
      const float2 v = make_float2(a, b), r = make_float2(inv, inv), t = __fmul2_rn(v, r);
      return __ffma2_rn(__ffma2_rn(t, make_float2(-unit, -unit), v), r, t);
    } else {
      const float t = a * inv, u = b * inv;
      return make_float2(fmaf(fmaf(-t, unit, a), inv, t), fmaf(fmaf(-u, unit, b), inv, u));
    }
  }
  template <bool PAIRS>
  __device__ __forceinline__ uint32_t four(const float *f) const {
    const float2 a = two<PAIRS>(f[0], f[1]), b = two<PAIRS>(f[2], f[3]);
    return pack_s8(__float2int_rn(a.x), __float2int_rn(a.y), __float2int_rn(b.x), __float2int_rn(b.y));
  }
};

// g / (1 + e^-g) * u, by e^-|g|: a denominator in [1, 2], for which the reciprocal instruction needs
// no care (the approximate quotient by one of 2^126 or more is 0, which is not what a large u makes of
// gates below -87), and e^-|g| as the square of a number that stays normal where it does not.
__device__ __forceinline__ float silu_mul(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fabsf(g) * -0.7213475204444817f));  // -log2(e) / 2
  e *= e;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return (g < 0.f ? g * e : g) * r * u;
}

// ---------------------------------------------------------------- rows in registers
// A group of G threads owns a row and holds it in registers, so the row is read once however
// many passes its statistics take: thread tid's i-th vector is 8 values, from (i G + tid) 8 on.
// Three layouts, told apart by where the rows lie in the 16-byte granules of memory:
//   kAligned  every row of every tensor starts at a granule and K is a multiple of 8
//   kSkewed   the tensors' rows start equally far into a granule (odd widths): vector j is
//             values 8 j - off .. 8 j - off + 7, whole granules but at a row's ends.  A group
//             only takes rows with one and the same off (their numbers differ by a multiple
//             of 8), so its columns stay put and their weights are loaded once.
//   kShifted  neither (the halves of SwiGLU rows of odd width): a vector is put together from
//             the granules that hold it
enum Layout { kAligned = 0, kSkewed = 1, kShifted = 2 };

template <typename T>
constexpr int kWords = 2 * (int)sizeof(T);  // 32-bit words of 8 values
template <typename T>
constexpr int kPerG = 16 / (int)sizeof(T);  // values per 16-byte granule

// A load of inputs.  Those of a kernel that is launched early are not constant over its run (its
// predecessor may still write them), so the read-only path, whose loads a compiler may move, is
// for the others.
template <bool CONST, typename V>
__device__ __forceinline__ V input(const V *p) {
  if constexpr (CONST)
    return __ldg(p);
  else
    return *p;
}

template <typename T>
__device__ __forceinline__ int misalign(const T *p) {  // values past a granule's start
  return (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
}

// c[i] = the words that start `off` values further on
template <typename T, int N>
__device__ __forceinline__ void shift_down(uint32_t (&c)[N], int off) {
  if constexpr (sizeof(T) == 2) {
    if (off & 4) {
#pragma unroll
      for (int i = 0; i + 2 < N; ++i) c[i] = c[i + 2];
    }
    if (off & 2) {
#pragma unroll
      for (int i = 0; i + 1 < N; ++i) c[i] = c[i + 1];
    }
    if (off & 1) {
#pragma unroll
      for (int i = 0; i + 1 < N; ++i) c[i] = __funnelshift_r(c[i], c[i + 1], 16);
    }
  } else {
    if (off & 2) {
#pragma unroll
      for (int i = 0; i + 2 < N; ++i) c[i] = c[i + 2];
    }
    if (off & 1) {
#pragma unroll
      for (int i = 0; i + 1 < N; ++i) c[i] = c[i + 1];
    }
  }
}

template <typename T>
__device__ __forceinline__ void words_to_floats(const uint32_t *u, float *f) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(u[i] << 16);
      f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(u[i]);
  }
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}
template <typename T>
__device__ __forceinline__ void floats_to_words(const float *f, uint32_t *u) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = pack2(f[2 * i], f[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(f[i]);
  }
}

// Eight values as they came from memory, unpacked where they are used so that many are in
// flight at once.
template <typename T, int LAYOUT, bool CONST = false>
struct Vec8 {
  static constexpr int N = kWords<T> + (LAYOUT == kShifted ? 4 : 0);
  uint32_t c[N];
  int off;

  template <int M>
  __device__ __forceinline__ void granules(const T *g) {
#pragma unroll
    for (int i = 0; i < M; i += 4) {
      const uint4 v = input<CONST>(reinterpret_cast<const uint4 *>(g) + i / 4);
      c[i] = v.x, c[i + 1] = v.y, c[i + 2] = v.z, c[i + 3] = v.w;
    }
  }
  __device__ __forceinline__ void singles(const T *p, int e, int K) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (e + k >= 0 && e + k < K) {
        if constexpr (sizeof(T) == 2)
          c[k / 2] |= (uint32_t)input<CONST>(reinterpret_cast<const uint16_t *>(p) + e + k) << (16 * (k & 1));
        else
          c[k] = input<CONST>(reinterpret_cast<const uint32_t *>(p) + e + k);
      }
  }
  // Values e .. e + 7 of the row p of K values, of a tensor whose values lie in [begin, end).
  // Granules that reach past the row's ends are read whole where they lie in the tensor (the
  // other values are dropped by unpack), so that no single loads are waited for.
  __device__ __forceinline__ void load(const T *p, int e, int K, const T *begin, const T *end) {
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = 0;
    if constexpr (LAYOUT == kAligned) {
      if (e < K) granules<N>(p + e);
    } else {
      const int row_off = LAYOUT == kShifted ? misalign(p) : 0;
      const T *g = p + e - row_off;
      off = row_off;
      if (e > -8 && e < K) {
        if (g >= begin && g + N * 4 / (int)sizeof(T) <= end) {
          granules<N>(g);
        } else {
          off = 0;
          singles(p, e, K);
        }
      }
    }
  }
  __device__ __forceinline__ void unpack(float *f, int e, int K) const {
    if constexpr (LAYOUT == kShifted) {
      uint32_t d[N];
#pragma unroll
      for (int i = 0; i < N; ++i) d[i] = c[i];
      shift_down<T>(d, off);
      words_to_floats<T>(d, f);
    } else {
      words_to_floats<T>(c, f);
    }
    if (LAYOUT != kAligned && (e < 0 || e + 8 > K)) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (e + k < 0 || e + k >= K) f[k] = 0.f;
    }
  }
};

// Stores values e .. e + 7 (those the row has).
template <typename T, int LAYOUT>
__device__ __forceinline__ void store8(T *p, int e, int K, const float *f) {
  if (LAYOUT == kAligned ? e < K : e >= 0 && e + 8 <= K) {
    uint32_t c[kWords<T>];
    floats_to_words<T>(f, c);
#pragma unroll
    for (int i = 0; i < kWords<T>; i += 4)
      reinterpret_cast<uint4 *>(p + e)[i / 4] = make_uint4(c[i], c[i + 1], c[i + 2], c[i + 3]);
  } else if (LAYOUT != kAligned && e < K) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (e + k >= 0 && e + k < K) p[e + k] = from_f<T>(f[k]);
  }
}

// weights e .. e + 7 (1 where there are none), put together from the granules that hold them;
// ALIGNED: they are a vector's, from a granule on
template <bool ALIGNED, typename W>
__device__ __forceinline__ void weights8_of(const W *w, int e, int K, float *f) {
  constexpr int N = kWords<W> + 4;
  const W *p = w + e;
  const int off = ALIGNED ? 0 : misalign(p);
  const W *g = p - off;
  uint32_t c[N];
  if (ALIGNED ? e < K : off == 0 && e >= 0 && e + 8 <= K) {
#pragma unroll
    for (int i = 0; i < N - 4; i += 4) {
      const uint4 v = reinterpret_cast<const uint4 *>(g)[i / 4];
      c[i] = v.x, c[i + 1] = v.y, c[i + 2] = v.z, c[i + 3] = v.w;
    }
    words_to_floats<W>(c, f);
  } else if (!ALIGNED && g >= w && g + N * 4 / (int)sizeof(W) <= w + K) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 v = reinterpret_cast<const uint4 *>(g)[i / 4];
      c[i] = v.x, c[i + 1] = v.y, c[i + 2] = v.z, c[i + 3] = v.w;
    }
    shift_down<W>(c, off);
    words_to_floats<W>(c, f);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = e + k >= 0 && e + k < K ? to_f<W>(w[e + k]) : 1.f;
  }
}
template <bool ALIGNED>
__device__ __forceinline__ void weights8(const void *w, int w_bf16, int e, int K, float *f) {
  if (!w) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = 1.f;
  } else if (w_bf16) {
    weights8_of<ALIGNED>(static_cast<const __nv_bfloat16 *>(w), e, K, f);
  } else {
    weights8_of<ALIGNED>(static_cast<const float *>(w), e, K, f);
  }
}

// A row's bytes, 8 per vector, to q (which starts at a multiple of 8 where `vec`).  Skewed vectors
// start `off` bytes before multiples of 8: they go through shared memory (`line`, 8 bytes per
// vector and 8 more), where the 8 bytes from 8 j on are 8 of a vector and the next one.
template <int VPT, int G, int LAYOUT>
__device__ __forceinline__ void store_bytes(int8_t *q, uint2 (&b)[VPT], uint2 *line, int off, int tid, int size, int K,
                                            bool vec) {
  if constexpr (LAYOUT == kSkewed) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) line[i * size + tid] = b[i];
    if constexpr (G == 32)
      __syncwarp();
    else
      __syncthreads();
    const int s = 8 * (off & 3);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const uint2 lo = line[i * size + tid], hi = line[i * size + tid + 1];
      const uint32_t c0 = off & 4 ? lo.y : lo.x, c1 = off & 4 ? hi.x : lo.y, c2 = off & 4 ? hi.y : hi.x;
      b[i] = make_uint2(__funnelshift_r(c0, c1, s), __funnelshift_r(c1, c2, s));
    }
    if constexpr (G == 32) __syncwarp();
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int e = (i * size + tid) * 8;
    if (LAYOUT == kAligned ? e < K : vec && e + 8 <= K) {
      *reinterpret_cast<uint2 *>(q + e) = b[i];
    } else if (LAYOUT != kAligned) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (e + k < K) q[e + k] = (int8_t)((k < 4 ? b[i].x : b[i].y) >> (8 * (k & 3)));
    }
  }
}

// Over the group: a warp, or the whole block of at most G threads.
template <int G>
__device__ __forceinline__ float group_sum(float v, float *red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (G > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const int warps = blockDim.x >> 5;
    v = 0.f;
#pragma unroll
    for (int i = 0; i < G / 32; ++i)
      if (i < warps) v += red[i];
  }
  return v;
}
template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v, uint32_t *red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (G > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const int warps = blockDim.x >> 5;
#pragma unroll
    for (int i = 0; i < G / 32; ++i)
      if (i < warps) v = max(v, red[i]);
  }
  return v;
}

constexpr int row_block(int G) { return G == 32 ? 256 : G; }  // (most) threads per block
// threads of the group this thread belongs to
template <int G>
__device__ __forceinline__ int group_size() {
  return G == 32 ? 32 : blockDim.x;
}

// What bounds it is the rows' one trip from and to HBM; see launch_width for the widths' groups
// and what they measured.
// Least blocks (of row_block(G) threads) per SM, which bounds the registers: 40 a thread for two
// vectors, 56 for four.  Only where that takes no spills (fp32 vectors and skewed rows' weights
// fill them).
template <typename T, int G, int VPT, int LAYOUT>
constexpr int row_blocks() {
  return sizeof(T) == 4 || LAYOUT != kAligned ? 0 : G == 512 ? 3 : G == 288 ? (VPT == 4 ? 4 : 5) : 0;
}
template <typename T, int MODE, int G, int VPT, int LAYOUT>
__global__ void __launch_bounds__(row_block(G), row_blocks<T, G, VPT, LAYOUT>()) row_kernel(const RowArgs a) {
  __shared__ float red_sum[2][32];
  __shared__ uint32_t red_max[2][32];
  constexpr int kPer = row_block(G) / G;  // rows of a block at a time
  __shared__ uint2 line[LAYOUT == kSkewed && MODE != kNorm ? kPer * (G * VPT + 1) : 1];
  constexpr bool kTwo = MODE != kQuantInt8;  // a second input: the residual, or SwiGLU's other half
  constexpr bool kIsNorm = MODE == kNorm || MODE == kNormInt8;
  race::wait_for_predecessor();
  race::let_successor_start();
  const int size = group_size<G>(), tid = G == 32 ? threadIdx.x % 32 : threadIdx.x, K = a.K;
  const long long first = (long long)blockIdx.x * kPer + (G == 32 ? threadIdx.x / 32 : 0);
  const long long step = LAYOUT == kSkewed ? (long long)gridDim.x * kPer : a.rows;
  const int off = LAYOUT == kSkewed ? misalign(static_cast<const T *>(a.x) + first * a.x_stride) : 0;
  auto at = [&](int i) { return (i * size + tid) * 8 - off; };  // where the thread's i-th vector starts
  float w[kIsNorm && LAYOUT == kSkewed ? VPT * 8 : 1];
  if constexpr (kIsNorm && LAYOUT == kSkewed) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) weights8<false>(a.w, a.w_bf16, at(i), K, w + 8 * i);
  }
  // the tensors' extents
  const T *x_begin = static_cast<const T *>(a.x), *x_end = x_begin + (a.rows - 1) * a.x_stride + (MODE == kSwigluInt8 ? 2 : 1) * (long long)K;
  const T *r_begin = MODE == kSwigluInt8 ? x_begin : static_cast<const T *>(a.r);
  const T *r_end = MODE == kSwigluInt8 ? x_end : r_begin + (a.rows - 1) * a.r_stride + K;
  int flip = 0;
  // (where a group is a block, the block's threads leave the loop together; else whole warps do)
  for (long long row = first; row < a.rows; row += step) {
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *r = MODE == kSwigluInt8 ? x + K : a.r ? static_cast<const T *>(a.r) + row * a.r_stride : nullptr;
    float v[VPT * 8];
    {
      Vec8<T, LAYOUT> vx[VPT], vr[VPT];
#pragma unroll
      for (int i = 0; i < VPT; ++i) vx[i].load(x, at(i), K, x_begin, x_end);
      if (kTwo && r) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) vr[i].load(r, at(i), K, r_begin, r_end);
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float *f = v + 8 * i;
        vx[i].unpack(f, at(i), K);
        if (kTwo && r) {
          float g[8];
          vr[i].unpack(g, at(i), K);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = MODE == kSwigluInt8 ? silu_mul(f[j], g[j]) : to_f<T>(from_f<T>(f[j] + g[j]));
          if (MODE != kSwigluInt8) store8<T, LAYOUT>(static_cast<T *>(a.h) + row * K, at(i), K, f);
        }
      }
    }

    if constexpr (kIsNorm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < VPT * 8; ++i) ss = fmaf(v[i], v[i], ss);
      const float rstd = rsqrtf(group_sum<G>(ss, red_sum[flip]) * a.inv_K + a.eps);
      if (a.rstd && tid == 0) a.rstd[row] = rstd;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float u[8];
        if (LAYOUT != kSkewed) weights8<LAYOUT == kAligned>(a.w, a.w_bf16, at(i), K, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[8 * i + j] = v[8 * i + j] * rstd * (LAYOUT == kSkewed ? w[kIsNorm && LAYOUT == kSkewed ? 8 * i + j : 0] : u[j]);
      }
    }
    if constexpr (MODE == kNorm) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) store8<T, LAYOUT>(static_cast<T *>(a.y) + row * K, at(i), K, v + 8 * i);
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < VPT * 8; ++i) m = max(m, abs_bits(v[i]));  // (0 past a row's ends)
      const Quantiser qz(group_max<G>(m, red_max[flip]));
      if (tid == 0) a.scale[row] = qz.scale;
      if (qz.lift != 1.f) {
#pragma unroll
        for (int i = 0; i < VPT * 8; ++i) v[i] = qz.lifted(v[i]);
      }
      int8_t *q = a.q + row * a.q_stride;
      uint2 b[VPT];
      // By pairs of values unless their registers cost a block per SM or spill (bf16: 8-bit norm of
      // 16384 x 8192 139 us by single values and 155 by pairs, rows of 16384 values to 8 bits 193
      // and 260; elsewhere 262144 x 256 to 8 bits 41 us by pairs and 42.5 by single values, 32768 x
      // 2048 37 and 38).
      constexpr bool kPairs = G < 1024 && !(MODE == kNormInt8 && VPT == 4);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        b[i] = make_uint2(qz.four<kPairs>(v + 8 * i), qz.four<kPairs>(v + 8 * i + 4));
      }
      store_bytes<VPT, G, LAYOUT>(q, b, line + (threadIdx.x / 32) * (G == 32 ? VPT * 32 + 1 : 0), off, tid, size, K, a.q_vec);
    }
    flip ^= 1;  // the next row's barrier lies between two uses of a half
  }
}

// Any width and any layout: the row is read again for each of its passes (from the caches), by
// single values.  What takes it is rows past the widths below, and a view beside dense tensors whose
// rows lie otherwise: 32768 x 2048 bf16 with x one value into its rows takes 133 us for the norm and
// 201 for the 8-bit norm, against 80 and 72 for aligned rows (64 rows: 3.6 and 4.2 against 1.9).
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
    const float v = value(i);
    q[i] = (int8_t)__float2int_rn(qz.two<false>(qz.lifted(v), 0.f).x);
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
  float inv_K = 0.f;
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

// A group of G threads walks rows; a thread keeps its columns' weights and sums of dw in
// registers over all of them, and has the next row's values on their way while it works on this
// one's where they are few or the group is a block (whose barrier every row pays): 200000 x 256
// bf16 124 us without, 105 with.
template <typename T, int G, int VPT, int LAYOUT>
__global__ void __launch_bounds__(row_block(G), G == 320 ? 2 : 512 / row_block(G)) bwd_kernel(const BwdArgs a) {
  constexpr int kPer = row_block(G) / G, N = VPT * 8;
  constexpr bool kAhead = G > 32 || VPT * sizeof(T) <= 4;  // (the registers of wider warps' rows would spill)
  __shared__ float red[2][32];
  extern __shared__ float warp_dw[];  // [groups of the block][K], where a block has several
  const int size = group_size<G>(), tid = G == 32 ? threadIdx.x % 32 : threadIdx.x, K = a.K;
  const int group = blockIdx.x * kPer + (G == 32 ? threadIdx.x / 32 : 0), groups = gridDim.x * kPer;
  const int off = LAYOUT == kSkewed ? misalign(static_cast<const T *>(a.dy) + (long long)group * K) : 0;
  auto at = [&](int i) { return (i * size + tid) * 8 - off; };  // where the thread's i-th vector starts
  float w[N], acc[N];
#pragma unroll
  for (int i = 0; i < VPT; ++i) weights8<false>(a.w, a.w_bf16, at(i), K, w + 8 * i);
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;

  struct Row {
    Vec8<T, LAYOUT, true> dy[VPT], h[VPT], dh[VPT];
    float rstd;
  };
  auto load = [&](Row &s, long long row) {
    const T *dy = static_cast<const T *>(a.dy) + row * K, *h = static_cast<const T *>(a.h) + row * K;
    const T *dh = a.dh ? static_cast<const T *>(a.dh) + row * K : nullptr;
    s.rstd = __ldg(a.rstd + row);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      s.dy[i].load(dy, at(i), K, dy - row * K, dy + (a.rows - row) * K);
      s.h[i].load(h, at(i), K, h - row * K, h + (a.rows - row) * K);
      if (dh) s.dh[i].load(dh, at(i), K, dh - row * K, dh + (a.rows - row) * K);
    }
  };
  int flip = 0;
  Row s;
  if (kAhead && group < a.rows) load(s, group);
  for (long long row = group; row < a.rows; row += groups) {
    Row next;
    if (kAhead) {
      if (row + groups < a.rows) load(next, row + groups);
    } else {
      load(s, row);
    }
    const float rstd = s.rstd;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float y[8], x[8];
      s.dy[i].unpack(y, at(i), K);
      s.h[i].unpack(x, at(i), K);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(y[j] * w[8 * i + j], x[j], sum);
    }
    const float c = group_sum<G>(sum, red[flip]) * rstd * rstd * a.inv_K;
    T *dx = static_cast<T *>(a.dx) + row * K;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float y[8], x[8], d[8];
      s.dy[i].unpack(y, at(i), K);
      s.h[i].unpack(x, at(i), K);
      if (a.dh) s.dh[i].unpack(d, at(i), K);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[8 * i + j] = fmaf(y[j], x[j] * rstd, acc[8 * i + j]);
        y[j] = rstd * fmaf(y[j], w[8 * i + j], -x[j] * c);
        if (a.dh) y[j] += d[j];
      }
      store8<T, LAYOUT>(dx, at(i), K, y);
    }
    flip ^= 1;  // a barrier of the next row lies between two uses of a half
    if (kAhead) s = next;
  }
  if (!a.part) return;
  float *part = a.part + (long long)blockIdx.x * K;
  float *mine = kPer == 1 ? part : warp_dw + (threadIdx.x / 32) * K;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at(i) + j >= 0 && at(i) + j < K) mine[at(i) + j] = acc[8 * i + j];
  if constexpr (kPer > 1) {
    __syncthreads();
    for (int c = threadIdx.x; c < K; c += row_block(G)) {
      float v = 0.f;
#pragma unroll
      for (int g = 0; g < kPer; ++g) v += warp_dw[g * K + c];
      part[c] = v;
    }
  }
}

// dw[k] = sum of the blocks' partial sums, in a fixed order.
__global__ void __launch_bounds__(1024) dw_sum_kernel(const float *part, int n, int K, void *dw, int w_bf16) {
  __shared__ float red[32][33];
  race::wait_for_predecessor();
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, k = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (k < K) {
#pragma unroll 4
    for (int i = g; i < n; i += 32) s += part[(long long)i * K + k];
  }
  red[g][lane] = s;
  __syncthreads();
  // transposed: warp g adds column g
  s = red[lane][g];
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int c = blockIdx.x * 32 + g;
  if (lane == 0 && c < K) {
    if (w_bf16)
      static_cast<__nv_bfloat16 *>(dw)[c] = __float2bfloat16_rn(s);
    else
      static_cast<float *>(dw)[c] = s;
  }
}

// Many rows of 8 bits back to values where granules are aligned on both sides: a thread takes the
// same granule of `out` in kDequantRows rows that follow one another, so that as many loads are on
// their way at once.  Bound by memory: 32768 x 2048 to bf16 in 31 us (6.5 TB/s), to fp32 in 52 us
// (6.4 TB/s); with the one row per thread of dequant_kernel 39 and 67 us, with rows blockDim.y
// apart 33 and 52 us (500000 x 128 to bf16: 40, 67 and 47 us).
constexpr int kDequantRows = 4;
template <typename T>
__global__ void __launch_bounds__(256) dequant_aligned_kernel(const int8_t *q, long long q_stride, const float *scale, T *out,
                                                              long long rows, int K) {
  constexpr int N = 16 / sizeof(T);  // values of a granule
  race::wait_for_predecessor();
  race::let_successor_start();
  const long long first = ((long long)blockIdx.x * blockDim.y + threadIdx.y) * kDequantRows;
  for (int e = threadIdx.x * N; e < K; e += blockDim.x * N) {
    uint32_t b[kDequantRows][N / 4];
    float s[kDequantRows];
#pragma unroll
    for (int r = 0; r < kDequantRows; ++r) {
      const long long row = first + r;
      if (row >= rows) continue;
      const uint32_t *p = reinterpret_cast<const uint32_t *>(q + row * q_stride + e);
      if constexpr (N == 8) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        b[r][0] = v.x, b[r][N / 4 - 1] = v.y;
      } else {
        b[r][0] = *p;
      }
      s[r] = scale[row];
    }
#pragma unroll
    for (int r = 0; r < kDequantRows; ++r) {
      const long long row = first + r;
      if (row >= rows) continue;
      float f[N];
#pragma unroll
      for (int k = 0; k < N; ++k) f[k] = (float)(int8_t)(b[r][k / 4] >> (8 * (k & 3))) * s[r];
      T *o = out + row * K + e;
      if constexpr (N == 8)
        store8<T, kAligned>(o - e, e, K, f);
      else
        *reinterpret_cast<float4 *>(o) = make_float4(f[0], f[1], f[2], f[3]);
    }
  }
}

// Rows of 8 bits back to values: a thread writes the 8 values of an output vector (a granule of
// bf16, two of fp32; skewed as the rows of `out` lie, see kSkewed), from the one or two aligned
// 8-byte words of q that hold their bytes.  blockDim.y rows per block.
template <typename T>
__global__ void __launch_bounds__(256) dequant_kernel(const int8_t *q_rows, long long q_stride, const float *scale, T *out,
                                                      long long rows, int K, bool q_vec) {
  race::wait_for_predecessor();
  race::let_successor_start();
  const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= rows) return;
  const float s = scale[row];
  const int8_t *q = q_rows + row * q_stride;
  T *o = out + row * K;
  const int off = misalign(o);
  for (int e = threadIdx.x * 8 - off; e < K; e += blockDim.x * 8) {
    const int w = e & ~7, shift = 8 * (e & 3);  // the word that holds byte e
    uint32_t lo = 0, hi = 0;
    if (q_vec && w >= 0 && w + (off ? 16 : 8) <= K) {
      const uint2 a = *reinterpret_cast<const uint2 *>(q + w);
      uint2 b = make_uint2(0, 0);
      if (off) b = *reinterpret_cast<const uint2 *>(q + w + 8);
      const bool half = e & 4;
      const uint32_t c0 = half ? a.y : a.x, c1 = half ? b.x : a.y, c2 = half ? b.y : b.x;
      lo = __funnelshift_r(c0, c1, shift);
      hi = __funnelshift_r(c1, c2, shift);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (e + k >= 0 && e + k < K) {
          const uint32_t v = (uint32_t)(uint8_t)q[e + k] << (8 * (k & 3));
          if (k < 4)
            lo |= v;
          else
            hi |= v;
        }
    }
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = (float)(int8_t)((k < 4 ? lo : hi) >> (8 * (k & 3))) * s;
    store8<T, kSkewed>(o, e, K, f);
  }
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

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Threads that `vectors` vectors at VPT per thread want: whole warps.
int threads_for(int vectors, int VPT) { return (vectors + 32 * VPT - 1) / (32 * VPT) * 32; }

template <typename T, int MODE, int G, int VPT, int LAYOUT>
void launch_row_kernel(const RowArgs &a, int vectors, cudaStream_t s) {
  constexpr int kPer = row_block(G) / G;
  const int threads = G == 32 ? row_block(G) : threads_for(vectors, VPT);
  long long blocks = (a.rows + kPer - 1) / kPer;
  if (LAYOUT == kSkewed) {
    // groups that walk rows, a multiple of 8 of them: as many as an SM's 2048 threads hold
    const long long most = 148 * (2048 / threads) / 8 * 8;
    blocks = blocks < most ? (blocks + 7) / 8 * 8 : most;
  }
  race::launch_early(row_kernel<T, MODE, G, VPT, LAYOUT>, dim3((unsigned)blocks), dim3(threads), 0, s, 1, a);
}

// Threads per row.  A warp up to 1024 values: no barriers, all of a row's loads in flight at
// once.  Wider rows take a block with two vectors per thread (32768 x 2048 bf16: norm 79 us with
// 128 threads, 83 with 64, 124 with a warp), four past 4096 values (8192: norm 157 us with 256
// threads, 171 with 512, 198 with 1024).  Their registers are bounded (see row_blocks) to what lets
// 48 warps onto an SM at 2048 values and 32 at 8192: before its quotients were exact the 8-bit norm of
// 32768 x 2048 took 80 us without that bound and 70 with it, of 16384 x 8192 169 and 136.  Few rows
// spread each over more threads, for latency.
template <typename T, int MODE, int LAYOUT>
void launch_width(const RowArgs &a, cudaStream_t s) {
  const int n = (a.K + (LAYOUT == kSkewed ? 7 : 0) + 7) / 8;  // vectors, whatever the offset
  const bool few = a.rows < 1184;  // eight blocks on each SM of a B200
  if (n <= 32) return launch_row_kernel<T, MODE, 32, 1, LAYOUT>(a, n, s);
  if (n <= 256 && few) return launch_row_kernel<T, MODE, 256, 1, LAYOUT>(a, n, s);
  if (n <= 64) return launch_row_kernel<T, MODE, 32, 2, LAYOUT>(a, n, s);
  if (n <= 96) return launch_row_kernel<T, MODE, 32, 3, LAYOUT>(a, n, s);
  if (n <= 128) return launch_row_kernel<T, MODE, 32, 4, LAYOUT>(a, n, s);
  if (n <= 576) return launch_row_kernel<T, MODE, 288, 2, LAYOUT>(a, n, s);
  if (n <= 1152 && LAYOUT != kAligned) return launch_row_kernel<T, MODE, 576, 2, LAYOUT>(a, n, s);
  if (n <= 1024 && few) return launch_row_kernel<T, MODE, 512, 2, LAYOUT>(a, n, s);
  if (n <= 1152) return launch_row_kernel<T, MODE, 288, 4, LAYOUT>(a, n, s);
  if (n <= 2048) return launch_row_kernel<T, MODE, 1024, 2, LAYOUT>(a, n, s);
  if constexpr (LAYOUT == kAligned) {
    if (n <= 4096) return launch_row_kernel<T, MODE, 1024, 4, LAYOUT>(a, n, s);
  }
  row_loop_kernel<T, MODE><<<(unsigned)a.rows, kNT, 0, s>>>(a);
}

// How far past a multiple of 16 bytes.
int past16(const void *p, int64_t bytes = 0) { return (int)((reinterpret_cast<uintptr_t>(p) + (uint64_t)bytes) & 15); }

template <typename T, int MODE>
void launch_type(RowArgs a, cudaStream_t s) {
  a.inv_K = 1.f / (float)a.K;
  const int64_t size = sizeof(T);
  a.q_vec = (reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)a.q_stride) % 8 == 0;
  if constexpr (MODE == kSwigluInt8) {
    if (a.K % 8 == 0 && aligned16(a.x) && past16(nullptr, a.x_stride * size) == 0 && a.q_vec)
      launch_width<T, MODE, kAligned>(a, s);
    else
      launch_width<T, MODE, kShifted>(a, s);
  } else {
    // whether the tensors' rows all start equally far into a granule: the first, and the step
    const int base = past16(a.x), step = past16(nullptr, a.x_stride * size), dense = past16(nullptr, a.K * size);
    bool alike = (!a.r || (past16(a.r) == base && past16(nullptr, a.r_stride * size) == step)) &&
                 (!(a.r || a.y) || dense == step) && (!a.y || past16(a.y) == base) && (!a.r || past16(a.h) == base);
    if (alike && base == 0 && step == 0 && a.K % 8 == 0 && aligned16(a.w) && a.q_vec)
      launch_width<T, MODE, kAligned>(a, s);
    else if (alike)
      launch_width<T, MODE, kSkewed>(a, s);
    else  // a view beside dense tensors, say
      row_loop_kernel<T, MODE><<<(unsigned)a.rows, kNT, 0, s>>>(a);
  }
}

template <int MODE>
int launch_rows(const char *what, const RowArgs &a, int dtype, cudaStream_t s) {
  if (dtype == RACE_BF16)
    launch_type<__nv_bfloat16, MODE>(a, s);
  else
    launch_type<float, MODE>(a, s);
  return launched(what);
}

// Blocks of the backward, each with one row of partial sums of dw to be added: four per SM of
// a B200, two where they hold eight rows at a time (up to 768 values), eight from there to 1024
// values (blocks of 64 threads where rows are aligned bf16, else of 128).  Few rows: as many blocks
// up to 148, 148 up to 592 rows, then one for four rows; blocks that hold eight rows at a time leave
// up to seven eighths of those without a row (1000 rows: 125 of 256 have some, the others add
// zeros).  A multiple of 8 (see kSkewed).
int bwd_blocks(int64_t rows, int64_t K) {
  const int64_t n = rows <= 148 ? rows : rows <= 592 ? 148 : (rows + 3) / 4, most = K <= 768 ? 296 : K <= 1024 ? 1184 : 592;
  return (int)(n < most ? (n + 7) / 8 * 8 : most);
}

template <typename T, int G, int VPT, int LAYOUT>
void launch_bwd_kernel(const BwdArgs &a, int blocks, int vectors, cudaStream_t s) {
  constexpr int kPer = row_block(G) / G;
  const int threads = G == 32 ? row_block(G) : threads_for(vectors, VPT);
  const size_t smem = a.part && kPer > 1 ? sizeof(float) * kPer * (size_t)a.K : 0;  // at most 24 KB
  bwd_kernel<T, G, VPT, LAYOUT><<<blocks, threads, smem, s>>>(a);
}

template <typename T, int LAYOUT>
void launch_bwd_width(const BwdArgs &a, int blocks, cudaStream_t s) {
  const int n = (a.K + (LAYOUT == kSkewed ? 7 : 0) + 7) / 8;
  if (n <= 32) return launch_bwd_kernel<T, 32, 1, LAYOUT>(a, blocks, n, s);
  if (n <= 64) return launch_bwd_kernel<T, 32, 2, LAYOUT>(a, blocks, n, s);
  if (n <= 96) return launch_bwd_kernel<T, 32, 3, LAYOUT>(a, blocks, n, s);
  // Two vectors per thread keep more bytes on their way (bf16, aligned: 65536 x 1024 101 us
  // against 134, 32768 x 2048 105 against 149); with fp32 or skewed rows they cost registers
  // that the blocks then lack (fp32 32768 x 2048 237 us against 168, bf16 65536 x 1001 196
  // against 138).
  // Blocks of 320 threads, two per SM, for 257 to 320 vectors: with those of 512, of which an SM's
  // registers hold one, fp32 20000 x 2047 takes 172 us against 131, 20000 x 2560 159 against 147,
  // 1000 x 2047 16.2 against 12.8, bf16 20000 x 2047 168 against 111.
  if constexpr (sizeof(T) == 2 && LAYOUT == kAligned) {
    if (n <= 128) return launch_bwd_kernel<T, 64, 2, LAYOUT>(a, blocks, n, s);
    if (n <= 256) return launch_bwd_kernel<T, 128, 2, LAYOUT>(a, blocks, n, s);
    if (n <= 512) return launch_bwd_kernel<T, 256, 2, LAYOUT>(a, blocks, n, s);
  }
  if (n <= 128) return launch_bwd_kernel<T, 128, 1, LAYOUT>(a, blocks, n, s);
  if (n <= 256) return launch_bwd_kernel<T, 256, 1, LAYOUT>(a, blocks, n, s);
  if (n <= 320) return launch_bwd_kernel<T, 320, 1, LAYOUT>(a, blocks, n, s);
  if (n <= 512) return launch_bwd_kernel<T, 512, 1, LAYOUT>(a, blocks, n, s);
  if (n <= 1024) return launch_bwd_kernel<T, 512, 2, LAYOUT>(a, blocks, n, s);
  if (n <= 2048) return launch_bwd_kernel<T, 512, 4, LAYOUT>(a, blocks, n, s);
  bwd_loop_kernel<T><<<blocks, kNT, 0, s>>>(a);
}

template <typename T>
void launch_bwd(BwdArgs a, int blocks, cudaStream_t s) {
  a.inv_K = 1.f / (float)a.K;
  const int base = past16(a.dy);
  const bool alike = past16(a.h) == base && past16(a.dx) == base && (!a.dh || past16(a.dh) == base);
  if (alike && base == 0 && a.K % 8 == 0)
    launch_bwd_width<T, kAligned>(a, blocks, s);
  else if (alike)
    launch_bwd_width<T, kSkewed>(a, blocks, s);
  else
    bwd_loop_kernel<T><<<blocks, kNT, 0, s>>>(a);
}

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
  const int size = value_size(dtype), w_size = weight ? value_size(weight_dtype) : 1;
  if (const int rc = check_values("race_rms_norm_fwd", {{x, size}, {residual, size}, {y, size}, {h, size}, {weight, w_size}, {rstd, 4}})) return rc;
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
  const int size = value_size(dtype), w_size = weight ? value_size(weight_dtype) : 1;
  if (const int rc = check_values("race_rms_norm_int8", {{x, size}, {residual, size}, {h, size}, {weight, w_size}, {scale, 4}})) return rc;
  RowArgs a{x, residual, weight, nullptr, h, q, scale, nullptr, rows, x_stride, residual_stride, q_stride, (int)K, weight_dtype == RACE_BF16, eps};
  return launch_rows<kNormInt8>("rms_norm_int8", a, dtype, reinterpret_cast<cudaStream_t>(stream));
}

int race_quant_int8(const void *x, int64_t x_stride, int dtype, int8_t *q, int64_t q_stride, float *scale, int64_t rows,
                    int64_t K, void *stream) {
  if (!x || !q || !scale) return err(RACE_ERR_ARG, "race_quant_int8: null pointer");
  if (const int rc = check_rows("race_quant_int8", rows, K, dtype)) return rc;
  if (x_stride < K || q_stride < K) return err(RACE_ERR_SHAPE, "race_quant_int8: row stride below the width %lld", K);
  if (const int rc = check_values("race_quant_int8", {{x, value_size(dtype)}, {scale, 4}})) return rc;
  RowArgs a{x, nullptr, nullptr, nullptr, nullptr, q, scale, nullptr, rows, x_stride, 0, q_stride, (int)K, 0, 0.f};
  return launch_rows<kQuantInt8>("quant_int8", a, dtype, reinterpret_cast<cudaStream_t>(stream));
}

int race_swiglu_int8(const void *gate_up, int64_t stride, int dtype, int8_t *q, int64_t q_stride, float *scale,
                     int64_t rows, int64_t F, void *stream) {
  if (!gate_up || !q || !scale) return err(RACE_ERR_ARG, "race_swiglu_int8: null pointer");
  if (const int rc = check_rows("race_swiglu_int8", rows, F, dtype)) return rc;
  if (stride < 2 * F || q_stride < F) return err(RACE_ERR_SHAPE, "race_swiglu_int8: row stride below the width (F=%lld)", F);
  if (const int rc = check_values("race_swiglu_int8", {{gate_up, value_size(dtype)}, {scale, 4}})) return rc;
  RowArgs a{gate_up, nullptr, nullptr, nullptr, nullptr, q, scale, nullptr, rows, stride, 0, q_stride, (int)F, 0, 0.f};
  return launch_rows<kSwigluInt8>("swiglu_int8", a, dtype, reinterpret_cast<cudaStream_t>(stream));
}

int race_dequant_int8(const int8_t *q, int64_t q_stride, const float *scale, void *out, int dtype, int64_t rows,
                      int64_t K, void *stream) {
  if (!q || !scale || !out) return err(RACE_ERR_ARG, "race_dequant_int8: null pointer");
  if (const int rc = check_rows("race_dequant_int8", rows, K, dtype)) return rc;
  if (q_stride < K) return err(RACE_ERR_SHAPE, "race_dequant_int8: row stride below the width %lld", K);
  if (const int rc = check_values("race_dequant_int8", {{out, value_size(dtype)}, {scale, 4}})) return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // rows of up to 2048 values share a block of 256 threads
  int x = 1;
  while (x < 256 && x * 8 < K + 7) x *= 2;
  const dim3 block((unsigned)x, (unsigned)(256 / x));
  unsigned grid = (unsigned)((rows + block.y - 1) / block.y);
  const bool q_vec = ((reinterpret_cast<uintptr_t>(q) | (uintptr_t)q_stride) & 7) == 0;
  // from 8 blocks per SM on (2400 x 2048 to bf16 3.3 -> 2.8 us, 1200 x 2048 2.15 -> 2.17 us); fewer
  // leave too few threads
  if (K % 8 == 0 && q_vec && aligned16(out) && grid >= 1184) {
    grid = (grid + kDequantRows - 1) / kDequantRows;
    if (dtype == RACE_BF16)
      race::launch_early(dequant_aligned_kernel<__nv_bfloat16>, dim3(grid), block, 0, s, 1, q, q_stride, scale,
                         static_cast<__nv_bfloat16 *>(out), rows, (int)K);
    else
      race::launch_early(dequant_aligned_kernel<float>, dim3(grid), block, 0, s, 1, q, q_stride, scale,
                         static_cast<float *>(out), rows, (int)K);
    return launched("dequant_int8");
  }
  if (dtype == RACE_BF16)
    race::launch_early(dequant_kernel<__nv_bfloat16>, dim3(grid), block, 0, s, 1, q, q_stride, scale,
                       static_cast<__nv_bfloat16 *>(out), rows, (int)K, q_vec);
  else
    race::launch_early(dequant_kernel<float>, dim3(grid), block, 0, s, 1, q, q_stride, scale, static_cast<float *>(out), rows,
                       (int)K, q_vec);
  return launched("dequant_int8");
}

size_t race_rms_norm_bwd_workspace_bytes(int64_t rows, int64_t K) {
  if (rows < 1 || K < 1) return 0;
  return sizeof(float) * (size_t)bwd_blocks(rows, K) * (size_t)K;
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
  const int size = value_size(dtype), w_size = weight || dw ? value_size(weight_dtype) : 1;
  if (const int rc = check_values("race_rms_norm_bwd", {{dy, size}, {dh, size}, {h, size}, {dx, size}, {rstd, 4}, {weight, w_size},
                                                        {dw, w_size}, {dw ? workspace : nullptr, 4}}))
    return rc;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int blocks = bwd_blocks(rows, K);
  BwdArgs a{dy, dh, h, weight, rstd, dx, dw, dw ? static_cast<float *>(workspace) : nullptr, rows, (int)K, weight_dtype == RACE_BF16};
  if (dtype == RACE_BF16)
    launch_bwd<__nv_bfloat16>(a, blocks, s);
  else
    launch_bwd<float>(a, blocks, s);
  if (const int rc = launched("rms_norm_bwd")) return rc;
  if (!dw) return RACE_OK;
  race::launch_early(dw_sum_kernel, dim3((unsigned)((K + 31) / 32)), dim3(1024), 0, s, 1, a.part, blocks, (int)K, dw,
                     (int)(weight_dtype == RACE_BF16));
  return launched("rms_norm_bwd dw");
}

}  // extern "C"
