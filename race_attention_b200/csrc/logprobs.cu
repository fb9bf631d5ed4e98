// logprobs.cu -- log probabilities of given tokens under rows of logits, with each
// row's entropy, its most probable entries, and the gradient.
//
// Mathematics, one row l of V logits, in base-2 logarithms: c = log2(e) / temperature,
//   d = (l - max(l)) c,  S = sum 2^d,  U = sum 2^d d
//   log2 p = d - log2 S,   entropy = (log2 S - U / S) ln 2
//   alternatives: the n largest l in the order (value descending, index ascending)
//   gradient for upstream a (of logp) and b (of the entropy):
//     dl = (a (1[token] - p) - b p (ln p + entropy)) / temperature
// max(l) and log2 S go to the backward as two numbers, and the difference is taken before the
// product with c: both keep the bits that tell a probability close to one from one, and a row
// that is masked with the type's lowest value throughout does not overflow.
//
// Entries of -infinity have probability 0 and add nothing.  A row of them alone has
// logp -infinity, entropy 0 and gradient 0.  A NaN in a row (or +infinity) makes its
// logp and entropy NaN; among the alternatives a NaN counts as -infinity.
#include "race_b200.h"

#include <math.h>

#include "common.cuh"
#include "internal.h"

namespace {

using race::err;
using race::from_f;
using race::launched;
using race::to_f;

constexpr int kNT = 512;
constexpr int kMaxTop = 32;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct FwdArgs {
  const void *logits;
  const int64_t *tokens;
  float *logp, *entropy, *top_logp;
  float2 *lse;
  int64_t *top_ids;
  long long stride, ignore;
  int V, n_top;
  float c, inv_temp;  // log2(e) / temperature, 1 / temperature
};

// Order of the alternatives as unsigned integers: value first (+-0 alike, NaN as
// -infinity), then the lower index.
__device__ __forceinline__ unsigned long long order_key(float l, int i) {
  if (l != l) l = -INFINITY;
  uint32_t b = __float_as_uint(l + 0.f);
  b = (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return ((unsigned long long)b << 32) | (0xffffffffu - (uint32_t)i);
}

template <typename F>
__device__ __forceinline__ float block_fold(float v, float *red, F f) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = red[0];
  for (int i = 1; i < (int)(blockDim.x >> 5); ++i) t = f(t, red[i]);
  return t;
}

template <typename T>
__global__ void __launch_bounds__(kNT) logprobs_fwd_kernel(FwdArgs a) {
  __shared__ float red[32];
  __shared__ unsigned long long keys[32];
  const long long row = blockIdx.x;
  const T *l = static_cast<const T *>(a.logits) + row * a.stride;
  const long long token = a.tokens[row];
  const int tid = threadIdx.x;
  if (token == a.ignore) {
    if (tid == 0) {
      a.logp[row] = 0.f;
      a.entropy[row] = 0.f;
      a.lse[row] = make_float2(0.f, 0.f);
    }
    if (tid < a.n_top) {
      a.top_ids[row * a.n_top + tid] = -1;
      a.top_logp[row * a.n_top + tid] = -INFINITY;
    }
    return;
  }
  float lm = -INFINITY;
  for (int i = tid; i < a.V; i += kNT) lm = fmaxf(lm, to_f<T>(l[i]));
  lm = block_fold(lm, red, [](float x, float y) { return fmaxf(x, y); });
  if (lm == -INFINITY) lm = 0.f;
  float s = 0.f, u = 0.f;
  for (int i = tid; i < a.V; i += kNT) {
    const float d = (to_f<T>(l[i]) - lm) * a.c;
    const float e = exp2f(d);
    s += e;
    u = fmaf(e, fmaxf(d, -200.f), u);  // 2^-200 is 0 in fp32; -infinity times it would be NaN
  }
  s = block_fold(s, red, [](float x, float y) { return x + y; });
  u = block_fold(u, red, [](float x, float y) { return x + y; });
  const bool empty = s == 0.f;
  const float log_s = empty ? -INFINITY : log2f(s);
  auto log_p = [&](int i) { return empty ? -INFINITY : (to_f<T>(l[i]) - lm) * a.inv_temp - log_s * kLn2; };
  if (tid == 0) {
    a.lse[row] = make_float2(lm, log_s);
    a.entropy[row] = empty ? 0.f : (log_s - u / s) * kLn2;
    a.logp[row] = token < 0 || token >= a.V ? NAN : log_p((int)token);
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.n_top; ++k) {
    unsigned long long best = 0;
    for (int i = tid; i < a.V; i += kNT) {
      const unsigned long long key = order_key(to_f<T>(l[i]), i);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if ((tid & 31) == 0) keys[tid >> 5] = best;
    __syncthreads();
    for (int i = 0; i < kNT / 32; ++i) best = max(best, keys[i]);
    last = best;
    if (tid == 0) {
      const int id = (int)(0xffffffffu - (uint32_t)best);
      a.top_ids[row * a.n_top + k] = id;
      a.top_logp[row * a.n_top + k] = log_p(id);
    }
  }
}

struct BwdArgs {
  const void *logits;
  const int64_t *tokens;
  const float2 *lse;
  const float *entropy, *g_logp, *g_entropy;
  void *dlogits;
  long long stride, ignore;
  int V;
  float c, inv_temp;
};

template <typename T>
__global__ void __launch_bounds__(kNT) logprobs_bwd_kernel(BwdArgs a) {
  const long long row = blockIdx.x;
  const T *l = static_cast<const T *>(a.logits) + row * a.stride;
  T *d = static_cast<T *>(a.dlogits) + row * a.V;
  const long long token = a.tokens[row];
  const float2 lse = a.lse[row];
  if (token == a.ignore || lse.y == -INFINITY) {
    for (int i = threadIdx.x; i < a.V; i += kNT) d[i] = from_f<T>(0.f);
    return;
  }
  const bool bad = token < 0 || token >= a.V;
  const float ga = bad ? NAN : a.g_logp ? a.g_logp[row] : 0.f, gb = a.g_entropy ? a.g_entropy[row] : 0.f;
  const float H = a.entropy[row];
  for (int i = threadIdx.x; i < a.V; i += kNT) {
    const float lq = fmaf(to_f<T>(l[i]) - lse.x, a.c, -lse.y);
    const float p = exp2f(lq);
    float v = -p * (ga + gb * fmaf(fmaxf(lq, -200.f), kLn2, H));
    if (i == token) v += ga;
    d[i] = from_f<T>(v * a.inv_temp);
  }
}

int check_shape(int64_t rows, int64_t V, int64_t stride, int dtype, float temperature) {
  if (dtype != RACE_F32 && dtype != RACE_BF16) return err(RACE_ERR_DTYPE, "token log probabilities: dtype %lld", dtype);
  if (rows < 1 || rows > 0x7fffffffLL || V < 1 || V > (1 << 30))
    return err(RACE_ERR_SHAPE, "token log probabilities: rows=%lld (1..2^31-1), vocabulary=%lld (1..2^30)", rows, V);
  if (stride < V) return err(RACE_ERR_SHAPE, "token log probabilities: row stride %lld below the vocabulary %lld", stride, V);
  if (!(temperature > 0.f) || isinf(temperature) || isinf(kLog2e / temperature))
    return err(RACE_ERR_ARG, "token log probabilities: the temperature must be positive and finite");
  return RACE_OK;
}

}  // namespace

extern "C" {

int race_token_logprobs_fwd(const void *logits, int64_t stride, int dtype, const int64_t *tokens, int64_t ignore_index,
                            float temperature, int n_top, float *logp, float *entropy, float *lse, int64_t *top_ids,
                            float *top_logp, int64_t rows, int64_t V, void *stream) {
  if (!logits || !tokens || !logp || !entropy || !lse || (n_top > 0 && (!top_ids || !top_logp)))
    return err(RACE_ERR_ARG, "race_token_logprobs_fwd: null pointer");
  if (reinterpret_cast<uintptr_t>(lse) & 7) return err(RACE_ERR_ALIGN, "race_token_logprobs_fwd: lse must be 8-byte aligned");
  if (const int rc = check_shape(rows, V, stride, dtype, temperature)) return rc;
  if (n_top < 0 || n_top > kMaxTop || n_top > V)
    return err(RACE_ERR_SHAPE, "race_token_logprobs_fwd: %lld alternatives (at most %lld, and the vocabulary)", n_top, kMaxTop);
  FwdArgs a{logits, tokens, logp, entropy, top_logp, reinterpret_cast<float2 *>(lse), top_ids, stride, ignore_index, (int)V, n_top,
            kLog2e / temperature, 1.f / temperature};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == RACE_BF16)
    logprobs_fwd_kernel<__nv_bfloat16><<<(unsigned)rows, kNT, 0, s>>>(a);
  else
    logprobs_fwd_kernel<float><<<(unsigned)rows, kNT, 0, s>>>(a);
  return launched("token_logprobs_fwd");
}

int race_token_logprobs_bwd(const void *logits, int64_t stride, int dtype, const int64_t *tokens, int64_t ignore_index,
                            float temperature, const float *lse, const float *entropy, const float *g_logp,
                            const float *g_entropy, void *dlogits, int64_t rows, int64_t V, void *stream) {
  if (!logits || !tokens || !lse || !entropy || !dlogits) return err(RACE_ERR_ARG, "race_token_logprobs_bwd: null pointer");
  if (reinterpret_cast<uintptr_t>(lse) & 7) return err(RACE_ERR_ALIGN, "race_token_logprobs_bwd: lse must be 8-byte aligned");
  if (const int rc = check_shape(rows, V, stride, dtype, temperature)) return rc;
  BwdArgs a{logits, tokens, reinterpret_cast<const float2 *>(lse), entropy, g_logp, g_entropy, dlogits, stride, ignore_index,
            (int)V, kLog2e / temperature, 1.f / temperature};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == RACE_BF16)
    logprobs_bwd_kernel<__nv_bfloat16><<<(unsigned)rows, kNT, 0, s>>>(a);
  else
    logprobs_bwd_kernel<float><<<(unsigned)rows, kNT, 0, s>>>(a);
  return launched("token_logprobs_bwd");
}

}  // extern "C"
