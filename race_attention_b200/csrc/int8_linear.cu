// int8_linear.cu -- product of 8-bit rows with 8-bit weight rows (a scale per token
// and per output channel) on the tcgen05 integer tensor cores.
//
// Mathematics: y[m, n] = (sum_k xq[m, k] wq[n, k]) * xs[m] * ws[n] + bias[n].  The sum is
// an exact 32-bit integer (widths up to 131071 cannot overflow it, even at -128 * -128);
// it is scaled in fp32 and rounded once to the output's type.
//
// One CTA computes a 128 x 128 tile: a producer lane streams 128-byte-wide K slices of
// both operands through a ring of shared-memory stages by TMA (rows and bytes past the
// tensors' ends read as 0, so ragged sizes need no special case), a second lane issues
// tcgen05.mma kind::i8 into a TMEM accumulator, and four warps scale and store it.
#include "race_b200.h"

#include <math.h>

#include <atomic>

#include "common.cuh"
#include "internal.h"
#include "tc_ptx.cuh"

namespace {

namespace tc = race::tc;
using race::cuda_err;
using race::err;

constexpr int kBM = 128, kBN = 128, kBK = 128;  // tile rows, channels, K bytes per stage
constexpr int kStages = 6;
constexpr int kThreads = 192;  // producer warp, MMA warp, four epilogue warps
constexpr int kABytes = kBM * kBK, kBBytes = kBN * kBK;
constexpr int kSmem = kStages * (kABytes + kBBytes) + 1024;
constexpr int kMaxDevices = 128;
constexpr int64_t kMaxK = 131071;  // 2^31 / 128^2, less one

// Set by a kernel whose bounded wait gave up (its outputs are NaN); read and cleared by
// calls made under race_set_status_check(1).
__device__ int g_timeout;

struct Args {
  const float *xs, *ws, *bias;
  void *y;
  long long M, N;
  int k_steps, vec_ok, withhold;
  uint32_t wait_limit;
};

// kind::i8: signed 8-bit operands, both K-major, 32-bit integer accumulator
constexpr uint32_t idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kThreads) int8_tile_kernel(const __grid_constant__ CUtensorMap mx,
                                                             const __grid_constant__ CUtensorMap mw, const Args a) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t full[kStages], empty[kStages], done;
  __shared__ uint32_t tmem_slot;
  __shared__ int ctl[2];  // {abort flag, poll limit}
  unsigned char *ring = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long m0 = (long long)blockIdx.y * kBM, n0 = (long long)blockIdx.x * kBN;
  volatile int *abort = ctl;

  if (threadIdx.x == 0) {
    ctl[0] = 0;
    ctl[1] = (int)a.wait_limit;
    for (int i = 0; i < kStages; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    tc::mbar_init(&done, 1);
    tc::fence_mbar_init();
  }
  if (warp == 1) tc::tmem_alloc(&tmem_slot, kBN);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == 0 && lane == 0) {
    int issued = 0;
    for (int k = 0; k < (a.withhold ? 0 : a.k_steps); ++k) {
      const int st = k % kStages, use = k / kStages;
      if (use && !tc::mbar_wait(&empty[st], (use - 1) & 1, abort)) break;
      unsigned char *sa = ring + st * (kABytes + kBBytes);
      tc::mbar_arrive_expect_tx(&full[st], kABytes + kBBytes);
      tc::tma_load_2d(sa, &mx, &full[st], k * kBK, (int)m0);
      tc::tma_load_2d(sa + kABytes, &mw, &full[st], k * kBK, (int)n0);
      issued = k + 1;
    }
    if (*abort)  // no copy may land after the block has gone
      for (int k = issued > kStages ? issued - kStages : 0; k < issued; ++k)
        tc::mbar_wait_drain(&full[k % kStages], (k / kStages) & 1);
  } else if (warp == 1 && lane == 0) {
    constexpr uint32_t id = idesc_i8(kBM, kBN);
    for (int k = 0; k < a.k_steps; ++k) {
      const int st = k % kStages;
      if (!tc::mbar_wait(&full[st], (k / kStages) & 1, abort)) break;
      tc::tc_fence_after();
      const uint32_t sa = tc::smem_u32(ring + st * (kABytes + kBBytes)), sb = sa + kABytes;
#pragma unroll
      for (int j = 0; j < kBK / 32; ++j)  // 32 bytes of K per instruction
        mma_i8(tmem, tc::sdesc(sa + 32 * j, 16, 1024), tc::sdesc(sb + 32 * j, 16, 1024), id, k | j);
      tc::mma_commit(&empty[st]);
    }
    tc::mma_commit(&done);
    if (*abort) tc::mbar_wait_drain(&done, 0);
  } else if (warp >= 2) {
    const int quarter = warp & 3;  // the TMEM lanes a warp may read
    const long long m = m0 + quarter * 32 + lane;
    const bool ok = tc::warp_all(tc::mbar_wait(&done, 0, abort) && !*abort);
    tc::tc_fence_after();
    const float xs = m < a.M ? a.xs[m] : 0.f;
    T *y = static_cast<T *>(a.y) + m * a.N;
    for (int c = 0; c < kBN; c += 32) {
      float v[32];
      tc::tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + c, v);
      tc::tmem_wait_ld();
      if (m < a.M) {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const long long n = n0 + c + j;
          if (n < a.N) {
            float f = (float)__float_as_int(v[j]) * xs * __ldg(a.ws + n);
            if (a.bias) f += __ldg(a.bias + n);
            y[n] = race::from_f<T>(ok ? f : NAN);
          }
        }
      }
      __syncwarp();  // TMEM loads are whole-warp instructions
    }
    if (!ok && lane == 0) atomicExch(&g_timeout, 1);
    tc::tc_fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, kBN);
  }
}

// Raises a kernel's dynamic shared-memory limit on the current device, once.
template <typename F>
cudaError_t allow_smem(F *kernel, int bytes, std::atomic<bool> (&set)[kMaxDevices]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (set[dev].load()) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) set[dev].store(true);
  return e;
}

template <typename T>
int launch(const CUtensorMap &mx, const CUtensorMap &mw, const Args &a, cudaStream_t s) {
  static std::atomic<bool> set[kMaxDevices];
  cudaError_t e = allow_smem(int8_tile_kernel<T>, kSmem, set);
  if (e != cudaSuccess) return cuda_err("int8_linear", e);
  const dim3 grid((unsigned)((a.N + kBN - 1) / kBN), (unsigned)((a.M + kBM - 1) / kBM));
  int8_tile_kernel<T><<<grid, kThreads, kSmem, s>>>(mx, mw, a);
  return race::launched("int8_linear");
}

// race_set_status_check(1): wait for the stream and report a wait that gave up.
int check_status(cudaStream_t s) {
  if (!race::status_check_on()) return RACE_OK;
  int flag = 0;
  cudaError_t e = cudaStreamSynchronize(s);
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&flag, g_timeout, sizeof(flag));
  if (e != cudaSuccess) return cuda_err("int8_linear", e);
  if (!flag) return RACE_OK;
  flag = 0;
  e = cudaMemcpyToSymbol(g_timeout, &flag, sizeof(flag));
  if (e != cudaSuccess) return cuda_err("int8_linear", e);
  return err(RACE_ERR_TIMEOUT, "int8_linear: a bounded wait expired");
}

}  // namespace

extern "C" {

int race_int8_linear(const int8_t *xq, int64_t x_stride, const float *x_scale, const int8_t *wq, int64_t w_stride,
                     const float *w_scale, const float *bias, void *y, int dtype, int64_t M, int64_t N, int64_t K,
                     void *stream) {
  if (!xq || !x_scale || !wq || !w_scale || !y) return err(RACE_ERR_ARG, "race_int8_linear: null pointer");
  if (dtype != RACE_F32 && dtype != RACE_BF16) return err(RACE_ERR_DTYPE, "race_int8_linear: dtype %lld", dtype);
  // the grid's second dimension holds M / 128
  if (M < 1 || N < 1 || M > 65535LL * kBM || N > 0x7fffff00LL)
    return err(RACE_ERR_SHAPE, "race_int8_linear: M=%lld or N=%lld out of range", M, N);
  if (K < 1 || K > kMaxK) return err(RACE_ERR_SHAPE, "race_int8_linear: K=%lld not in 1..%lld", K, kMaxK);
  if (x_stride < K || w_stride < K) return err(RACE_ERR_SHAPE, "race_int8_linear: row stride below K=%lld", K);
  if (((reinterpret_cast<uintptr_t>(xq) | reinterpret_cast<uintptr_t>(wq) | (uintptr_t)x_stride | (uintptr_t)w_stride) & 15) ||
      ((reinterpret_cast<uintptr_t>(x_scale) | reinterpret_cast<uintptr_t>(w_scale) | reinterpret_cast<uintptr_t>(bias)) & 3))
    return err(RACE_ERR_ALIGN, "race_int8_linear: 8-bit rows must start at multiples of 16 bytes");
  CUtensorMap mx, mw;
  if (!race::make_byte_rows_map(&mx, xq, M, K, x_stride, kBM) || !race::make_byte_rows_map(&mw, wq, N, K, w_stride, kBN))
    return err(RACE_ERR_CUDA, "race_int8_linear: no tensor map for M=%lld, N=%lld", M, N);
  Args a{x_scale, w_scale, bias, y, M, N, (int)((K + kBK - 1) / kBK), 0, race::withhold_first_load() ? 1 : 0,
         race::current_wait_limit()};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int rc = dtype == RACE_BF16 ? launch<__nv_bfloat16>(mx, mw, a, s) : launch<float>(mx, mw, a, s);
  return rc == RACE_OK ? check_status(s) : rc;
}

}  // extern "C"
