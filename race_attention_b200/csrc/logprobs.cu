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
//
// The forward reads a row once, by a block or (few rows) a cluster of up to 8 blocks with a
// share each: every thread keeps its running maximum, S and U, and where its maximum lies, and
// the threads' are joined at the end.  The alternatives need no second pass over the row: the
// n-th largest of the threads' maxima (or of groups of four threads) bounds the n-th largest
// entry from below, and only the few threads whose maximum reaches it hold candidates, whose
// entries are read again from the L2 cache.
#include "race_b200.h"

#include <math.h>

#include "common.cuh"
#include "internal.h"

namespace {

using race::err;
using race::from_f;
using race::launched;
using race::to_f;

constexpr int kMaxTop = 32;
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct FwdArgs {
  const void *logits;
  const int64_t *tokens;
  float *logp, *entropy, *top_logp;
  float2 *lse;
  int64_t *top_ids;
  long long stride, ignore, rows;
  int V, n_top;
  float c, inv_temp;  // log2(e) / temperature, 1 / temperature
};

// 2^x (2 units in the last place; 0 below 2^-126)
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Order of the alternatives as unsigned integers: value first (+-0 alike, NaN as
// -infinity), then the lower index.
__device__ __forceinline__ unsigned long long order_key(float l, int i) {
  if (l != l) l = -INFINITY;
  uint32_t b = __float_as_uint(l + 0.f);
  b = (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return ((unsigned long long)b << 32) | (0xffffffffu - (uint32_t)i);
}

__device__ __forceinline__ float key_value(unsigned long long key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float((b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int key_index(unsigned long long key) { return (int)(0xffffffffu - (uint32_t)key); }

template <typename T>
constexpr int kPer = 16 / (int)sizeof(T);  // logits per 16-byte granule

template <typename T>
__device__ __forceinline__ int misalign(const T *p) {
  return (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4 &v, float (&f)[kPer<T>]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      f[2 * i] = __uint_as_float(u[i] << 16);
      f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    } else {
      f[i] = __uint_as_float(u[i]);
    }
  }
}

// A row of V logits as 16-byte granules: granule j holds entries kPer j - off and on; the first
// and the last may reach past the row, into its neighbours or out of [begin, end).
template <typename T>
struct RowView {
  const T *row, *begin, *end;
  int V, off;
  __device__ __forceinline__ RowView(const void *logits, long long r, long long stride, long long rows, int v)
      : row(static_cast<const T *>(logits) + r * stride),
        begin(static_cast<const T *>(logits)),
        end(begin + (rows - 1) * stride + v),
        V(v),
        off(misalign(row)) {}
  __device__ __forceinline__ int granules() const { return (V + off + kPer<T> - 1) / kPer<T>; }
  __device__ __forceinline__ int first(int j) const { return j * kPer<T> - off; }
  // its entries, -infinity in the places of those the row does not have
  __device__ __forceinline__ uint4 load(int j) const {
    const int e = first(j);
    const T *g = row + e;
    uint4 v;
    if (e >= 0 && e + kPer<T> <= V) {
      v = *reinterpret_cast<const uint4 *>(g);
    } else {
      uint32_t u[4];
      const bool whole = g >= begin && g + kPer<T> <= end;
      if (whole) v = *reinterpret_cast<const uint4 *>(g);
      u[0] = v.x, u[1] = v.y, u[2] = v.z, u[3] = v.w;
#pragma unroll
      for (int k = 0; k < kPer<T>; ++k) {
        const bool has = e + k >= 0 && e + k < V;
        if constexpr (sizeof(T) == 2) {
          const int s = 16 * (k & 1);
          uint32_t x = 0xff80u;
          if (has) x = whole ? (u[k / 2] >> s) & 0xffffu : (uint32_t)reinterpret_cast<const uint16_t *>(g)[k];
          u[k / 2] = (u[k / 2] & (0xffff0000u >> s)) | (x << s);
        } else {
          if (!has)
            u[k] = 0xff800000u;
          else if (!whole)
            u[k] = reinterpret_cast<const uint32_t *>(g)[k];
        }
      }
      v = make_uint4(u[0], u[1], u[2], u[3]);
    }
    return v;
  }
};

// largest entry of a granule (a NaN only if there is nothing else)
template <typename T>
__device__ __forceinline__ float granule_max(const uint4 &v) {
  if constexpr (sizeof(T) == 2) {
    const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&v);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  } else {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
}

// Running statistics: the largest logit (-infinity: none yet, taken as 0), and S and U relative
// to it.
struct Stat {
  float m, s, u;
  // the same relative to a larger maximum
  __device__ __forceinline__ void rebase(float to, float c) {
    const float d = m == -INFINITY ? 0.f : (m - (to == -INFINITY ? 0.f : to)) * c;
    const float k = exp2f(d);
    u = k * fmaf(s, fmaxf(d, -200.f), u);
    s *= k;
    m = to;
  }
  // those of the whole warp, in every lane
  __device__ __forceinline__ void join_warp(float c) {
    float to = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, o));
    rebase(to, c);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      u += __shfl_xor_sync(0xffffffffu, u, o);
    }
  }
};

// ---- clusters
__device__ __forceinline__ uint32_t smem_u32(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// What the blocks of a row's cluster send its first one.
struct Shared {
  Stat stat[kMaxCluster];
  unsigned long long top[kMaxCluster * kMaxTop];
};

// Grid: C blocks (a cluster) per row; block `rank` of a row takes its granules [G rank / C,
// G (rank + 1) / C), thread t those at t, t + kNT, ... of them, kBatch on their way at a time.
template <typename T, int kNT>
__global__ void __launch_bounds__(kNT) logprobs_fwd_kernel(const FwdArgs a, const int C) {
  // (with the next batch on its way: 8192 x 50257 bf16 takes 168 us in batches of one granule, 141
  // of two, 148 of four, and 285 without)
  constexpr int kBatch = 2, kWarps = kNT / 32;
  constexpr int kCandidates = kNT == 32 ? 256 : 1024;  // entries at or above the bound that are ranked at once
  __shared__ Shared sh;
  __shared__ Stat warp_stat[kWarps];
  __shared__ unsigned long long bound[kNT], cand[kCandidates], tau;
  __shared__ int n_owner, n_cand, owner[kNT];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x % C;
  const long long row = blockIdx.x / C;
  race::wait_for_predecessor();
  race::let_successor_start();
  const long long token = a.tokens[row];
  if (token == a.ignore) {  // the whole cluster leaves
    if (rank == 0 && tid == 0) {
      a.logp[row] = 0.f;
      a.entropy[row] = 0.f;
      if (a.lse) a.lse[row] = make_float2(0.f, 0.f);
    }
    if (rank == 0 && tid < a.n_top) {
      a.top_ids[row * a.n_top + tid] = -1;
      a.top_logp[row * a.n_top + tid] = -INFINITY;
    }
    return;
  }
  if (C > 1) cluster_arrive();  // this block runs
  const RowView<T> view(a.logits, row, a.stride, a.rows, a.V);
  const int G = view.granules();
  const int g0 = (int)((long long)G * rank / C), g1 = (int)((long long)G * (rank + 1) / C);

  // ---- one pass: maximum, S, U, and the granule that holds the thread's first maximum
  Stat st = {-INFINITY, 0.f, 0.f};
  int best = g0 + tid;
  const float2 c2 = make_float2(a.c, a.c);
  auto absorb = [&](auto &v, int j) {  // granules j, j + kNT, ... of the thread
    constexpr int n = sizeof(v) / sizeof(uint4);
    float gm[n], bm = -INFINITY;
#pragma unroll
    for (int b = 0; b < n; ++b) {
      gm[b] = granule_max<T>(v[b]);
      bm = fmaxf(bm, gm[b]);
    }
    if (bm > st.m) {
#pragma unroll
      for (int b = n - 1; b >= 0; --b)
        if (gm[b] == bm) best = j + b * kNT;
      st.rebase(bm, a.c);
    }
    const float m = st.m == -INFINITY ? 0.f : st.m;
    const float2 m2 = make_float2(-m, -m);
    float2 s2 = make_float2(0.f, 0.f), u2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int b = 0; b < n; ++b) {
      float f[kPer<T>];
      unpack<T>(v[b], f);
#pragma unroll
      for (int k = 0; k < kPer<T>; k += 2) {
        float2 d = __fmul2_rn(__fadd2_rn(make_float2(f[k], f[k + 1]), m2), c2);
        const float2 e = make_float2(exp2_approx(d.x), exp2_approx(d.y));
        d.x = fmaxf(d.x, -200.f);  // 2^-200 is 0 in fp32; -infinity times it would be NaN
        d.y = fmaxf(d.y, -200.f);
        s2 = __fadd2_rn(s2, e);
        u2 = __ffma2_rn(e, d, u2);
      }
    }
    st.s += s2.x + s2.y;
    st.u += u2.x + u2.y;
  };
  // The row's whole granules; the next batch is on its way while this one is worked on.
  const int whole0 = view.off ? 1 : 0, whole1 = (a.V + view.off) / kPer<T>;
  const int w1 = min(g1, whole1);
  int j = g0 + tid;
  if (j < whole0) {  // (a first granule with some of the row: one thread's)
    const uint4 v[1] = {view.load(j)};
    absorb(v, j);
    j += kNT;
  }
  const uint4 *base = reinterpret_cast<const uint4 *>(view.row - view.off);
  uint4 v[kBatch];
  if (j + (kBatch - 1) * kNT < w1) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) v[b] = base[j + b * kNT];
    for (; j + (2 * kBatch - 1) * kNT < w1; j += kBatch * kNT) {
      uint4 next[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) next[b] = base[j + (kBatch + b) * kNT];
      absorb(v, j);
#pragma unroll
      for (int b = 0; b < kBatch; ++b) v[b] = next[b];
    }
    absorb(v, j);
    j += kBatch * kNT;
  }
  for (; j < g1; j += kNT) {
    const uint4 one[1] = {j < w1 ? base[j] : view.load(j)};
    absorb(one, j);
  }
  const float thread_max = st.m;
  st.join_warp(a.c);
  if (lane == 0) warp_stat[warp] = st;

  // ---- alternatives of this block's share: candidates are what reaches tau
  const bool top = a.n_top > 0;
  unsigned long long mine = 0;  // 0: no entries
  // threads whose joint maximum enters the bound: four where that leaves more than 32 of them
  // with entries (fewer keys to rank), else one
  constexpr int kGroup = kNT >= 256 ? 4 : 1;
  const int group = g1 - g0 >= kNT ? kGroup : 1, n_keys = kNT / group;
  if (top) {
    // upper end of the granule: an index no lower than the first maximum's
    if (g0 + tid < g1) mine = order_key(thread_max, view.first(best) + kPer<T> - 1);
    unsigned long long k = mine;
    if (group == 4) {
      k = max(k, __shfl_xor_sync(0xffffffffu, k, 1));
      k = max(k, __shfl_xor_sync(0xffffffffu, k, 2));
    }
    if (tid % group == 0) bound[tid / group] = k;
    if (tid == 0) n_owner = n_cand = 0, tau = 0;
  }
  __syncthreads();
  if (warp == 0) {
    st = lane < kWarps ? warp_stat[lane] : Stat{-INFINITY, 0.f, 0.f};
    st.join_warp(a.c);
    if (lane == 0) sh.stat[rank] = st;
  }
  if (top) {
    if (tid < n_keys) {
      const unsigned long long k = bound[tid];
      int above = 0;
#pragma unroll 8
      for (int i = 0; i < n_keys; ++i) above += bound[i] > k;
      if (k && above == a.n_top - 1) tau = k;  // (keys of groups with entries differ)
    }
    __syncthreads();
    const unsigned long long t = tau;
    auto offer = [&](int j) {  // a granule's entries that reach the bound
      const uint4 v = view.load(j);
      float f[kPer<T>];
      unpack<T>(v, f);
#pragma unroll
      for (int k = 0; k < kPer<T>; ++k) {
        const int e = view.first(j) + k;
        const unsigned long long key = order_key(f[k], e);
        if (key >= t && e >= 0 && e < a.V) {
          const int n = atomicAdd(&n_cand, 1);
          if (n < kCandidates) cand[n] = key;
        }
      }
    };
    if (mine && mine >= t) owner[atomicAdd(&n_owner, 1)] = tid;
    __syncthreads();
    // the owners' granules, dealt out to all threads
    const int each = (g1 - g0 + kNT - 1) / kNT, items = n_owner * each;
    for (int i = tid; i < items; i += kNT) {
      const int j = g0 + owner[i / each] + i % each * kNT;
      if (j < g1) offer(j);
    }
    __syncthreads();
    const int n = n_cand;
    unsigned long long *out = sh.top + rank * a.n_top;
    if (n <= kCandidates) {
      // (n_top places, of which a block with fewer entries leaves the last ones 0)
      for (int i = tid; i < a.n_top; i += kNT)
        if (i >= n) out[i] = 0;
      for (int i = tid; i < n; i += kNT) {
        const unsigned long long k = cand[i];
        int above = 0;
#pragma unroll 8
        for (int q = 0; q < n; ++q) above += cand[q] > k;
        if (above < a.n_top) out[above] = k;
      }
    } else {
      // more entries reach the bound than fit (a few threads that hold most of the large ones, or
      // chance: about 1 % of rows of 4000 random bf16 values with 32 alternatives): one pass of
      // the share for each alternative
      unsigned long long last = ~0ull;
      for (int i = 0; i < a.n_top; ++i) {
        unsigned long long k = 0;
        for (int j = g0 + tid; j < g1; j += kNT) {
          const uint4 v = view.load(j);
          float f[kPer<T>];
          unpack<T>(v, f);
#pragma unroll
          for (int q = 0; q < kPer<T>; ++q) {
            const int e = view.first(j) + q;
            const unsigned long long x = order_key(f[q], e);
            if (e >= 0 && e < a.V && x < last && x > k) k = x;
          }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
        __syncthreads();
        if (lane == 0) bound[warp] = k;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) k = max(k, bound[w]);
        last = k;
        if (tid == 0) out[i] = k;
      }
    }
  }

  // ---- the cluster's shares go to its first block
  if (C > 1) {
    if (top) __syncthreads();
    cluster_wait();
    if (rank) {
      if (tid == 0) {
        const uint32_t to = map_rank(smem_u32(&sh.stat[rank]), 0);
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(st.m) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(st.s) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(st.u) : "memory");
      }
      if (tid < a.n_top)
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(map_rank(smem_u32(&sh.top[rank * a.n_top + tid]), 0)),
                     "l"(sh.top[rank * a.n_top + tid])
                     : "memory");
    }
    cluster_arrive();
    cluster_wait();
    if (rank) return;
  } else if (top) {
    __syncthreads();
  }
  if (C == 1 && !top && warp) return;

  // ---- the row's results
  Stat all = st;  // (in warp 0, the only one with C == 1 and no alternatives, every lane's)
  if (C > 1 || top) {
    all = lane < C ? sh.stat[lane] : Stat{-INFINITY, 0.f, 0.f};
    all.join_warp(a.c);
  }
  const bool empty = all.s == 0.f;
  const float lm = all.m == -INFINITY ? 0.f : all.m, log_s = empty ? -INFINITY : log2f(all.s);
  auto log_p = [&](float l) { return empty ? -INFINITY : (l - lm) * a.inv_temp - log_s * kLn2; };
  if (tid == 0) {
    if (a.lse) a.lse[row] = make_float2(lm, log_s);
    const float entropy = empty ? 0.f : (log_s - all.u / all.s) * kLn2;
    a.entropy[row] = entropy < 0.f ? 0.f : entropy;  // (rounding; a NaN stays)
    a.logp[row] = token < 0 || token >= a.V ? NAN : log_p(to_f<T>(view.row[token]));
  }
  const int n = C * a.n_top;
  for (int i = tid; i < n; i += kNT) {
    const unsigned long long k = sh.top[i];
    int place = i;
    if (C > 1) {
      place = 0;
#pragma unroll 8
      for (int q = 0; q < n; ++q) place += sh.top[q] > k;
    }
    if (k && place < a.n_top) {
      a.top_ids[row * a.n_top + place] = key_index(k);
      // (a NaN ranks as -infinity, and its row's S is NaN)
      a.top_logp[row * a.n_top + place] = log_p(key_value(k));
    }
  }
}

struct BwdArgs {
  const void *logits;
  const int64_t *tokens;
  const float2 *lse;
  const float *entropy, *g_logp, *g_entropy;
  void *dlogits;
  long long stride, ignore, rows;
  int V;
  float c, inv_temp;
};

// What a row's gradient needs: dl = p (A + B log2 p), and `one` more at the token.
struct RowGrad {
  float lm, log_s, A, B, one;
  bool zero;
  long long token;
  __device__ __forceinline__ RowGrad(const BwdArgs &a, long long row) {
    token = a.tokens[row];
    const float2 lse = a.lse[row];
    lm = lse.x, log_s = lse.y;
    zero = token == a.ignore || log_s == -INFINITY;
    const bool bad = token < 0 || token >= a.V;
    const float up = a.g_logp ? a.g_logp[row] : 0.f, gb = a.g_entropy ? a.g_entropy[row] : 0.f;
    const float ga = bad && up != 0.f ? NAN : up;  // (a logp that is not used has gradient 0, NaN or not)
    A = -(ga + gb * a.entropy[row]) * a.inv_temp;
    B = -gb * kLn2 * a.inv_temp;
    one = ga * a.inv_temp;
  }
};

// Rows of logits and gradient that start equally far into a granule (dense ones do): 16-byte
// accesses but at a row's ends.  Grid (rows, shares of a row).
template <typename T, bool ENTROPY, int kNT>
__global__ void __launch_bounds__(kNT) logprobs_bwd_kernel(const BwdArgs a) {
  constexpr int kBatch = 2;  // (8192 x 50257 bf16: 272 us with one, 261 with two, 254 with four, which lose on short rows)
  race::wait_for_predecessor();
  race::let_successor_start();
  const long long row = blockIdx.x;
  const RowGrad g(a, row);
  const RowView<T> view(a.logits, row, a.stride, a.rows, a.V);
  T *d = static_cast<T *>(a.dlogits) + row * a.V;
  const int G = view.granules(), C = gridDim.y;
  const int g0 = (int)((long long)G * blockIdx.y / C), g1 = (int)((long long)G * (blockIdx.y + 1) / C);
  const float2 m2 = make_float2(-g.lm, -g.lm), c2 = make_float2(a.c, a.c), s2 = make_float2(-g.log_s, -g.log_s);
  const float2 A2 = make_float2(g.A, g.A), B2 = make_float2(g.B, g.B);
  // where the token's entry lies, counted from the first granule's start
  const int token_at = g.token >= 0 && g.token < a.V ? (int)g.token + view.off : -1;

  auto gradient = [&](const uint4 &v, int j, float(&f)[kPer<T>]) {
    unpack<T>(v, f);
#pragma unroll
    for (int k = 0; k < kPer<T>; k += 2) {
      float2 q = __ffma2_rn(__fadd2_rn(make_float2(f[k], f[k + 1]), m2), c2, s2);  // log2 p
      const float2 p = make_float2(exp2_approx(q.x), exp2_approx(q.y));
      float2 w = A2;
      if (ENTROPY) {
        q.x = fmaxf(q.x, -200.f);  // p is 0 there, and -infinity times it would be NaN
        q.y = fmaxf(q.y, -200.f);
        w = __ffma2_rn(B2, q, A2);
      }
      w = __fmul2_rn(p, w);
      f[k] = w.x, f[k + 1] = w.y;
    }
    if (token_at >= j * kPer<T> && token_at < (j + 1) * kPer<T>) {
#pragma unroll
      for (int k = 0; k < kPer<T>; ++k)
        if (token_at == j * kPer<T> + k) f[k] += g.one;
    }
  };
  const uint4 *from = reinterpret_cast<const uint4 *>(view.row - view.off);
  uint4 *to = reinterpret_cast<uint4 *>(d - view.off);
  auto whole = [&](const uint4 &v, int j) {
    float f[kPer<T>];
    gradient(v, j, f);
    uint4 o;
    if constexpr (sizeof(T) == 2) {
      uint32_t u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
        u[k] = *reinterpret_cast<const uint32_t *>(&h);
      }
      o = make_uint4(u[0], u[1], u[2], u[3]);
    } else {
      o = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
    to[j] = o;
  };
  auto part = [&](int j) {  // a granule that the row has some of
    float f[kPer<T>];
    if (g.zero) {
#pragma unroll
      for (int k = 0; k < kPer<T>; ++k) f[k] = 0.f;
    } else {
      gradient(view.load(j), j, f);
    }
    const int e = view.first(j);
#pragma unroll
    for (int k = 0; k < kPer<T>; ++k)
      if (e + k >= 0 && e + k < a.V) d[e + k] = from_f<T>(f[k]);
  };

  const int whole0 = view.off ? 1 : 0, w1 = min(g1, (a.V + view.off) / kPer<T>);
  int j = g0 + threadIdx.x;
  if (j < whole0) {
    part(j);
    j += kNT;
  }
  if (g.zero) {
    for (; j < w1; j += kNT) to[j] = make_uint4(0, 0, 0, 0);
  } else if (j + (kBatch - 1) * kNT < w1) {
    // the next batch is on its way while this one is worked on
    uint4 v[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) v[b] = from[j + b * kNT];
    for (; j + (2 * kBatch - 1) * kNT < w1; j += kBatch * kNT) {
      uint4 next[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) next[b] = from[j + (kBatch + b) * kNT];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        whole(v[b], j + b * kNT);
        v[b] = next[b];
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) whole(v[b], j + b * kNT);
    j += kBatch * kNT;
  }
  for (; j < g1; j += kNT)
    if (j < w1)
      whole(from[j], j);
    else
      part(j);
}

// Any layout, one value at a time.
template <typename T, int kNT>
__global__ void __launch_bounds__(kNT) logprobs_bwd_loop_kernel(const BwdArgs a) {
  race::wait_for_predecessor();
  race::let_successor_start();
  const long long row = blockIdx.x;
  const RowGrad g(a, row);
  const T *l = static_cast<const T *>(a.logits) + row * a.stride;
  T *d = static_cast<T *>(a.dlogits) + row * a.V;
  for (int i = blockIdx.y * kNT + threadIdx.x; i < a.V; i += gridDim.y * kNT) {
    float v = 0.f;
    if (!g.zero) {
      const float q = fmaf(to_f<T>(l[i]) - g.lm, a.c, -g.log_s);
      v = exp2_approx(q) * fmaf(g.B, fmaxf(q, -200.f), g.A);
      if (i == g.token) v += g.one;
    }
    d[i] = from_f<T>(v);
  }
}

template <typename T, int kNT>
int launch_fwd_threads(const FwdArgs &a, cudaStream_t s) {
  // Blocks per row: more while there are fewer than four blocks on each SM of a B200 and every
  // thread still has a granule.
  int C = 1;
  if (kNT == 256)
    while (C < kMaxCluster && a.rows * C * 2 <= 4 * 148 && a.V >= 2 * C * kNT * kPer<T>) C *= 2;
  const cudaError_t e =
      race::launch_early(logprobs_fwd_kernel<T, kNT>, dim3((unsigned)(a.rows * C)), dim3(kNT), 0, s, (unsigned)C, a, C);
  if (e != cudaSuccess) return race::cuda_err("token_logprobs_fwd", e);
  return launched("token_logprobs_fwd");
}

template <typename T>
int launch_fwd(const FwdArgs &a, cudaStream_t s) {
  // A row's fixed work (its joins) is per warp: few threads for short rows (8192 rows of 4000
  // bf16 values: 29 us with 32 threads, 34 with 128; of 10000: 66 with 128, 84 with 256).
  const int granules = (a.V + kPer<T> - 1) / kPer<T>;
  if (granules <= 512) return launch_fwd_threads<T, 32>(a, s);
  if (granules <= 2048) return launch_fwd_threads<T, 128>(a, s);
  return launch_fwd_threads<T, 256>(a, s);
}

template <typename T, int kNT>
int launch_bwd_threads(const BwdArgs &a, cudaStream_t s) {
  // shares of a row: sixteen blocks' worth on each SM of a B200 while a thread has two granules
  long long C = 1;
  while (a.rows * C < 16 * 148 && a.V >= 4 * C * kNT * kPer<T>) C *= 2;
  const dim3 grid((unsigned)a.rows, (unsigned)C);
  const uintptr_t l = reinterpret_cast<uintptr_t>(a.logits), d = reinterpret_cast<uintptr_t>(a.dlogits);
  if (((l ^ d) & 15) == 0 && (a.stride - a.V) % kPer<T> == 0) {
    if (a.g_entropy)
      race::launch_early(logprobs_bwd_kernel<T, true, kNT>, grid, dim3(kNT), 0, s, 1, a);
    else
      race::launch_early(logprobs_bwd_kernel<T, false, kNT>, grid, dim3(kNT), 0, s, 1, a);
  } else {
    race::launch_early(logprobs_bwd_loop_kernel<T, kNT>, grid, dim3(kNT), 0, s, 1, a);
  }
  return launched("token_logprobs_bwd");
}

template <typename T>
int launch_bwd(const BwdArgs &a, cudaStream_t s) {
  return (a.V + kPer<T> - 1) / kPer<T> <= 512 ? launch_bwd_threads<T, 64>(a, s) : launch_bwd_threads<T, 256>(a, s);
}

int check_shape(int64_t rows, int64_t V, int64_t stride, int dtype, float temperature) {
  if (dtype != RACE_F32 && dtype != RACE_BF16) return err(RACE_ERR_DTYPE, "token log probabilities: dtype %lld", dtype);
  // granules are numbered, and candidates' keys hold indexes, in 32 bits; a grid has 2^31 - 1 rows
  if (rows < 1 || rows > 0x7fffffffLL || V < 1 || V > (1 << 28))
    return err(RACE_ERR_SHAPE, "token log probabilities: rows=%lld (1..2^31-1), vocabulary=%lld (1..2^28)", rows, V);
  if (stride < V)
    return err(RACE_ERR_SHAPE, "token log probabilities: row stride %lld below the vocabulary %lld", stride, V);
  if (!(temperature > 0.f) || isinf(temperature) || isinf(kLog2e / temperature))
    return err(RACE_ERR_ARG, "token log probabilities: the temperature must be positive and finite");
  return RACE_OK;
}

}  // namespace

extern "C" {

int race_token_logprobs_fwd(const void *logits, int64_t stride, int dtype, const int64_t *tokens, int64_t ignore_index,
                            float temperature, int n_top, float *logp, float *entropy, float *lse, int64_t *top_ids,
                            float *top_logp, int64_t rows, int64_t V, void *stream) {
  if (!logits || !tokens || !logp || !entropy || (n_top > 0 && (!top_ids || !top_logp)))
    return err(RACE_ERR_ARG, "race_token_logprobs_fwd: null pointer");
  if (reinterpret_cast<uintptr_t>(lse) & 7) return err(RACE_ERR_ALIGN, "race_token_logprobs_fwd: lse must be 8-byte aligned");
  if (const int rc = check_shape(rows, V, stride, dtype, temperature)) return rc;
  if (n_top < 0 || n_top > kMaxTop || n_top > V)
    return err(RACE_ERR_SHAPE, "race_token_logprobs_fwd: %lld alternatives (at most %lld, and the vocabulary)", n_top, kMaxTop);
  if (const int rc = race::check_values("race_token_logprobs_fwd", {{logits, race::value_size(dtype)}, {tokens, 8}, {logp, 4}, {entropy, 4},
                                                                    {n_top ? top_ids : nullptr, 8}, {n_top ? top_logp : nullptr, 4}}))
    return rc;
  FwdArgs a{logits, tokens, logp, entropy, top_logp, reinterpret_cast<float2 *>(lse), top_ids, stride, ignore_index, rows, (int)V, n_top,
            kLog2e / temperature, 1.f / temperature};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == RACE_BF16 ? launch_fwd<__nv_bfloat16>(a, s) : launch_fwd<float>(a, s);
}

int race_token_logprobs_bwd(const void *logits, int64_t stride, int dtype, const int64_t *tokens, int64_t ignore_index,
                            float temperature, const float *lse, const float *entropy, const float *g_logp,
                            const float *g_entropy, void *dlogits, int64_t rows, int64_t V, void *stream) {
  if (!logits || !tokens || !lse || !entropy || !dlogits) return err(RACE_ERR_ARG, "race_token_logprobs_bwd: null pointer");
  if (reinterpret_cast<uintptr_t>(lse) & 7) return err(RACE_ERR_ALIGN, "race_token_logprobs_bwd: lse must be 8-byte aligned");
  if (const int rc = check_shape(rows, V, stride, dtype, temperature)) return rc;
  const int size = race::value_size(dtype);
  if (const int rc = race::check_values("race_token_logprobs_bwd", {{logits, size}, {dlogits, size}, {tokens, 8}, {entropy, 4}, {g_logp, 4},
                                                                    {g_entropy, 4}}))
    return rc;
  BwdArgs a{logits, tokens, reinterpret_cast<const float2 *>(lse), entropy, g_logp, g_entropy, dlogits, stride, ignore_index,
            rows, (int)V, kLog2e / temperature, 1.f / temperature};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return dtype == RACE_BF16 ? launch_bwd<__nv_bfloat16>(a, s) : launch_bwd<float>(a, s);
}

}  // extern "C"
