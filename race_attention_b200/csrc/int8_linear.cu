// int8_linear.cu -- product of 8-bit rows with 8-bit weight rows (a scale per token
// and per output channel) on the tcgen05 integer tensor cores.
//
// Mathematics: y[m, n] = (sum_k xq[m, k] wq[n, k]) * xs[m] * ws[n] + bias[n].  The sum is
// an exact 32-bit integer (widths up to 131071 cannot overflow it, even at -128 * -128), in
// whatever order its parts are added; it is scaled in fp32 and rounded once to the output's
// type.
//
// Operands come in as 128-byte-wide K slices by TMA (128-byte swizzle), through a ring of
// shared-memory stages; rows and bytes past the tensors' ends read as 0, so ragged sizes need
// no special case.  One lane issues the copies, one the tcgen05.mma kind::i8, and four warps
// scale and store the accumulators they read from TMEM.  Two kernels share that scheme:
//
// * split_kernel, for few tokens: the weights are the MMA's rows (128 channels per CTA), the
//   tokens its columns (16 to 128), so a weight byte is read once and the tensor cores idle
//   under a stream of weights.  Up to 8 CTAs of a cluster share a tile's K range and add their
//   integer sums through each other's shared memory, which gives every SM weights to stream
//   when the layer has few channels, with no workspace and no atomics.
// * pair_kernel, for many: a pair of CTAs computes 256 tokens x 256 channels with
//   cta_group::2 (each SM holds half of either operand), persistent over the tiles, with two
//   accumulators in TMEM so that one tile's stores overlap the next one's products.
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

constexpr int kBK = 128;                  // K bytes per stage (one swizzled row)
constexpr int kTileRows = 128;            // operand rows per tile and CTA
constexpr int kTileBytes = kTileRows * kBK;
constexpr int kThreads = 192;             // producer warp, MMA warp, four epilogue warps
constexpr int kMaxDevices = 128;
constexpr int64_t kMaxK = 131071;         // 2^31 / 128^2, less one
constexpr int kMaxSplit = 8;              // CTAs of a cluster that share a tile's K range

// Set by a kernel whose bounded wait gave up (its outputs are NaN); read and cleared by
// calls made under race_set_status_check(1).
__device__ int g_timeout;

struct Args {
  const float *xs, *ws, *bias;
  void *y;
  int M, N, k_steps;
  int m_tiles, n_tiles;  // pair_kernel
  int vec_ok;            // output rows start at multiples of 16 bytes
  int withhold;
  uint32_t wait_limit;
};

// kind::i8: signed 8-bit operands, both K-major, 32-bit integer accumulator
constexpr uint32_t idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

template <int CG>
__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}

// One stage's products: 128 bytes of K in steps of 32 (2 in a descriptor's address field,
// which holds 16-byte units and does not carry: stages start at multiples of 1024).
template <int CG>
__device__ __forceinline__ void mma_stage(uint32_t d_tmem, uint32_t sa, uint32_t sb, uint32_t idesc, bool first) {
  const uint64_t da = tc::sdesc(sa, 16, 1024), db = tc::sdesc(sb, 16, 1024);
#pragma unroll
  for (int j = 0; j < kBK / 32; ++j) mma_i8<CG>(d_tmem, da + 2 * j, db + 2 * j, idesc, !(first && j == 0));
}

// ---- cluster helpers
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_rank(uint32_t smem_addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
  return r;
}
// every thread of every CTA of the cluster
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}
__device__ __forceinline__ void st_cluster_i(uint32_t addr, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ int ld_cluster_i(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// ---- a pair of CTAs (cta_group::2)
// Tile load into this CTA's shared memory that completes on the pair leader's barrier.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap *map, uint32_t leader_bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(leader_bar)
      : "memory");
}
// One arrival on the barrier at this offset in both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void commit_pair(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(tc::smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t *dst, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(dst)), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t addr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(ncols) : "memory");
}

__device__ __forceinline__ unsigned char *align_1k(unsigned char *p) {
  return reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(p) + 1023) & ~(uintptr_t)1023);
}

// ------------------------------------------------------------------ few tokens
template <int BT>
struct Split {
  static constexpr int kStageBytes = kTileBytes + BT * kBK;
  // 72 to 128 KB on the way into a CTA; two CTAs per SM up to 64 tokens
  static constexpr int kStages = BT <= 16 ? 5 : BT <= 32 ? 4 : BT <= 64 ? 3 : 4;
  static constexpr int kRing = kStages * kStageBytes;
  static constexpr int kBytes = kRing + BT * kTileRows * 4 + 1024;
  static constexpr int kCols = BT < 32 ? 32 : BT;  // TMEM columns (a power of two of at least 32)
};

// Grid (S * channel tiles, token tiles), clusters of S along x: rank r of a cluster takes the
// r-th S-th of the K steps, and stores channels [r, r + 1) * 128 / S of the tile, to whose sums
// every rank sends its part.
template <typename T, int BT>
__global__ void __launch_bounds__(kThreads) split_kernel(const __grid_constant__ CUtensorMap mx,
                                                         const __grid_constant__ CUtensorMap mw, const Args a, const int S) {
  using C = Split<BT>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t full[C::kStages], empty[C::kStages], done;
  __shared__ uint32_t tmem_slot;
  __shared__ int ctl[2];  // {abort flag, poll limit}
  __shared__ int bad;     // some rank's sums are missing
  __shared__ float xs[BT];
  unsigned char *ring = align_1k(smem_raw);
  // [rank][token][channel of this CTA] integer sums
  int *sums = reinterpret_cast<int *>(ring + C::kRing);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % S, n0 = (int)(blockIdx.x / S) * kTileRows, m0 = blockIdx.y * BT;
  const int width = kTileRows / S;  // channels this CTA stores: 16 to 128
  const int tokens = min(BT, a.M - m0);
  const int k_begin = (int)((long long)a.k_steps * rank / S), k_end = (int)((long long)a.k_steps * (rank + 1) / S);
  const int steps = k_end - k_begin;
  volatile int *abort = ctl;

  // The producer lane sets the barriers up and has the first copies on their way before the
  // rest of the block is ready.
  int st = 0, issued = 0;
  uint32_t parity = 1;  // a fresh barrier's last phase counts as done
  auto load_next = [&]() {
    unsigned char *sw = ring + st * C::kStageBytes;
    tc::mbar_arrive_expect_tx(&full[st], C::kStageBytes);
    tc::tma_load_2d(sw, &mw, &full[st], (k_begin + issued) * kBK, n0);
    tc::tma_load_2d(sw + kTileBytes, &mx, &full[st], (k_begin + issued) * kBK, m0);
    ++issued;
    if (++st == C::kStages) st = 0, parity ^= 1;
  };
  const int wanted = a.withhold ? 0 : steps;
  if (threadIdx.x == 64) {
    tc::prefetch_tmap(&mx);
    tc::prefetch_tmap(&mw);
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    tc::mbar_init(&done, 1);
    ctl[0] = 0;
    ctl[1] = (int)a.wait_limit;
    bad = 0;
    tc::fence_mbar_init();
    race::wait_for_predecessor();
    while (issued < wanted && issued < C::kStages) load_next();
  }
  if (warp == 1) tc::tmem_alloc(&tmem_slot, C::kCols);
  race::wait_for_predecessor();
  for (int t = (int)threadIdx.x - 64; t < tokens; t += kThreads - 64)
    if (t >= 0) xs[t] = a.xs[m0 + t];
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  race::let_successor_start();  // (this block has its shared memory and TMEM)
  if (S > 1) cluster_arrive();  // this block runs, and its `bad` is clear

  if (warp == 0) {
    if (lane == 0) {
      while (issued < wanted) {
        if (!tc::mbar_wait(&empty[st], parity, abort)) break;
        load_next();
      }
      // No copy may land after the block has gone, whether or not this thread learns that another
      // one has given up (waiting for them costs nothing: the products wait for the same).
      for (int k = issued > C::kStages ? issued - C::kStages : 0; k < issued; ++k)
        tc::mbar_wait_drain(&full[k % C::kStages], (k / C::kStages) & 1);
    }
    __syncwarp();
    if (S > 1) cluster_wait();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t id = idesc_i8(kTileRows, BT);
      int at = 0;
      uint32_t phase = 0;
      bool ready = false;  // as in pair_kernel: the next stage's wait runs behind this one's issue
      for (int k = 0; k < steps; ++k) {
        if (!ready && !tc::mbar_wait(&full[at], phase, abort)) break;
        tc::tc_fence_after();
        const int now = at;
        if (++at == C::kStages) at = 0, phase ^= 1;
        ready = tc::mbar_try_wait(&full[at], phase);
        const uint32_t sw = tc::smem_u32(ring) + now * C::kStageBytes;
        mma_stage<1>(tmem, sw, sw + kTileBytes, id, k == 0);
        tc::mma_commit(&empty[now]);
      }
      if (*abort) __threadfence_block();  // (who sees `done` sees that it was given up)
      tc::mma_commit(&done);
      tc::mbar_wait_drain(&done, 0);  // no product may be under way when the block goes, either
    }
    __syncwarp();
    if (S > 1) cluster_wait();
  } else {
    // send this rank's sums to the blocks that store them: a thread has one channel
    const int quarter = warp & 3;  // the TMEM lanes a warp may read
    const int c = quarter * 32 + lane, owner = c / width;
    if (S > 1) cluster_wait();
    const bool ok = tc::warp_all(tc::mbar_wait(&done, 0, abort) && !*abort);
    tc::tc_fence_after();
    const uint32_t to = map_rank(tc::smem_u32(sums + (rank * BT) * width + c - owner * width), owner);
    const uint32_t row = 4 * width;
#pragma unroll
    for (int t0 = 0; t0 < BT; t0 += 16) {
      if (t0 < tokens) {
        float v[16];
        tc::tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + t0, v);
        tc::tmem_wait_ld();
#pragma unroll
        for (int t = 0; t < 16; ++t)
          if (t0 + t < tokens) st_cluster_i(to + (t0 + t) * row, __float_as_int(v[t]));
      }
    }
    if (!ok && lane < S) st_cluster_i(map_rank(tc::smem_u32(&bad), lane), 1);
    tc::tc_fence_before();
    __syncwarp();
  }
  if (S > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }

  // add the ranks' sums, scale and store: a thread has four channels and every `step`-th token
  const bool ok = *(volatile int *)&bad == 0;
  const int quads = width / 4, q = threadIdx.x % quads, step = kThreads / quads;
  const int n = n0 + rank * width + 4 * q;
  if (n < a.N) {
    float ws[4], bias[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int nn = min(n + j, a.N - 1);
      ws[j] = a.ws[nn];
      bias[j] = a.bias ? a.bias[nn] : 0.f;
    }
    T *y = static_cast<T *>(a.y) + (long long)m0 * a.N + n;
#pragma unroll 4
    for (int t = threadIdx.x / quads; t < tokens; t += step) {
      const int4 *from = reinterpret_cast<const int4 *>(sums + t * width + 4 * q);
      int4 acc = from[0];
#pragma unroll
      for (int r = 1; r < kMaxSplit; ++r)
        if (r < S) {
          const int4 v = from[r * (BT * width / 4)];
          acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
        }
      const float s = xs[t];
      float f[4] = {fmaf((float)acc.x * s, ws[0], bias[0]), fmaf((float)acc.y * s, ws[1], bias[1]),
                    fmaf((float)acc.z * s, ws[2], bias[2]), fmaf((float)acc.w * s, ws[3], bias[3])};
      if (!ok) f[0] = f[1] = f[2] = f[3] = NAN;
      T *o = y + (long long)t * a.N;
      if (a.vec_ok) {  // N is a multiple of 16 bytes' worth of values: n + 3 < N too
        if constexpr (sizeof(T) == 2)
          *reinterpret_cast<uint2 *>(o) = make_uint2(tc::pack_bf16(f[0], f[1]), tc::pack_bf16(f[2], f[3]));
        else
          *reinterpret_cast<float4 *>(o) = make_float4(f[0], f[1], f[2], f[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < a.N) o[j] = race::from_f<T>(f[j]);
      }
    }
  }
  if (!ok && threadIdx.x == 0) atomicExch(&g_timeout, 1);
  if (warp == 1) {
    __syncwarp();
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, C::kCols);
  }
}

// ------------------------------------------------------------------ many tokens
constexpr int kPairStages = 6;
constexpr int kPairStageBytes = 2 * kTileBytes;
constexpr int kPairN = 256;               // channels per tile and accumulator columns
constexpr int kOutWarps = 8;              // epilogue warps: two per TMEM lane quarter, half of the columns each
constexpr int kPairThreads = 64 + 32 * kOutWarps;
// One arrival on this CTA's barrier once the pair's MMAs issued so far are done.
__device__ __forceinline__ void commit_leader(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}

// everything the pair kernel keeps in shared memory (227 KB per CTA allow one more kilobyte)
struct PairSmem {
  unsigned char ring[kPairStages][kPairStageBytes];
  unsigned char out[kOutWarps][32 * 128];  // 32 rows x 128 bytes on their way out
  float scale[kPairN], bias[kPairN];       // of the tile's channels
  uint64_t full[kPairStages], empty[kPairStages], acc_full[2], acc_empty[2], drained;
  uint32_t tmem_slot;
  int ctl[2];   // {abort flag, poll limit}
  int filled;   // stages this CTA has asked for
  int gave_up;  // a wait of either CTA has
};
constexpr int kGroupM = 8;                // token tiles that share their weight tiles in L2

// The t-th tile: groups of kGroupM token tiles, inside a group the token tile varies fastest.
__device__ __forceinline__ void tile_at(const Args &a, int t, int &mt, int &nt) {
  const int group = t / (kGroupM * a.n_tiles);
  const int in = t - group * (kGroupM * a.n_tiles);
  const int gm = min(kGroupM, a.m_tiles - group * kGroupM);
  nt = in / gm;
  mt = group * kGroupM + in - nt * gm;
}

template <typename T>
__global__ void __launch_bounds__(kPairThreads) __cluster_dims__(2, 1, 1)
pair_kernel(const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mw, const Args a) {
  extern __shared__ __align__(1024) unsigned char pair_smem[];
  PairSmem &sm = *reinterpret_cast<PairSmem *>(pair_smem);
  uint64_t *full = sm.full, *empty = sm.empty, *acc_full = sm.acc_full, *acc_empty = sm.acc_empty;
  unsigned char *ring = sm.ring[0];
  float *scale = sm.scale, *bias = sm.bias;
  int *ctl = sm.ctl;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = a.m_tiles * a.n_tiles;
  volatile int *abort = ctl;

  if (threadIdx.x == 0) {
    tc::prefetch_tmap(&mx);
    tc::prefetch_tmap(&mw);
    ctl[0] = (tc::smem_u32(ring) & 1023) != 0;  // the swizzled tiles start at multiples of 1024
    ctl[1] = (int)a.wait_limit;
    sm.filled = sm.gave_up = 0;
    for (int i = 0; i < kPairStages; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&acc_full[i], 1);
      tc::mbar_init(&acc_empty[i], 2 * kOutWarps);  // the pair's epilogue warps
    }
    tc::mbar_init(&sm.drained, 1);
    tc::fence_mbar_init();
  }
  if (warp == 1) tmem_alloc_pair(&sm.tmem_slot, 2 * kPairN);
  tc::tc_fence_before();
  cluster_sync();  // both CTAs' barriers exist
  tc::tc_fence_after();
  const uint32_t tmem = sm.tmem_slot;

  if (warp == 0) {
    if (lane == 0 && !a.withhold) {
      int st = 0, filled = 0;     // the next stage, and how many were asked for
      uint32_t parity = 1;        // of the wait for a free stage: a fresh barrier's last phase counts as done
      bool go = true, ready = true;
      const uint32_t leader_full = map_rank(tc::smem_u32(&full[0]), 0);
      for (int t = pair; go && t < tiles; t += pairs) {
        int mt, nt;
        tile_at(a, t, mt, nt);
        const int m = mt * 256 + rank * kTileRows, n = nt * kPairN + rank * kTileRows;
        for (int k = 0; k < a.k_steps; ++k) {
          if (!ready && !tc::mbar_wait(&empty[st], parity, abort)) {
            go = false;
            break;
          }
          const int now = st;
          if (++st == kPairStages) st = 0, parity ^= 1;
          ready = tc::mbar_try_wait(&empty[st], parity);  // answers while this stage's copies are issued
          const uint32_t sa = tc::smem_u32(ring) + now * kPairStageBytes;
          const uint32_t bar = leader_full + now * 8;
          // the leader's barrier counts both CTAs' bytes; the peer's may land first
          if (rank == 0) tc::mbar_arrive_expect_tx(&full[now], 2 * kPairStageBytes);
          tma_load_pair(sa, &mx, bar, k * kBK, m);
          tma_load_pair(sa + kTileBytes, &mw, bar, k * kBK, n);
          ++filled;
        }
      }
      sm.filled = filled;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t id = idesc_i8(256, kPairN);
      int st = 0, buf = 0;
      uint32_t parity = 0, acc_parity = 1;
      // Even on a completed barrier a wait answers only after some 300 cycles, so each asks for
      // the next stage before it issues this one's work: 410 -> 355 us at 8192^3 (827 -> 650
      // cycles per stage on this thread, of which the products take 512).
      bool go = true, ready = false;
      for (int t = pair; go && t < tiles; t += pairs) {
        if (!tc::mbar_wait(&acc_empty[buf], acc_parity, abort)) break;
        tc::tc_fence_after();
        for (int k = 0; k < a.k_steps; ++k) {
          if (!ready && !tc::mbar_wait(&full[st], parity, abort)) {
            go = false;
            break;
          }
          tc::tc_fence_after();
          const int now = st;
          if (++st == kPairStages) st = 0, parity ^= 1;
          ready = tc::mbar_try_wait(&full[st], parity);
          const uint32_t sa = tc::smem_u32(ring) + now * kPairStageBytes;
          mma_stage<2>(tmem + buf * kPairN, sa, sa + kTileBytes, id, k == 0);
          commit_pair(&empty[now]);
        }
        if (go) commit_pair(&acc_full[buf]);
        if (++buf == 2) buf = 0, acc_parity ^= 1;
      }
      commit_leader(&sm.drained);  // no product may be under way when the CTAs go
      tc::mbar_wait_drain(&sm.drained, 0);
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;  // the TMEM lanes a warp may read; its columns
    const int et = threadIdx.x - 64;                       // over the epilogue warps
    const uint32_t stage = tc::smem_u32(sm.out[warp - 2]);
    constexpr int kCols = 128 / (int)sizeof(T);  // columns per 128-byte output row
    int i = 0;
    for (int t = pair; t < tiles; t += pairs, ++i) {
      int mt, nt;
      tile_at(a, t, mt, nt);
      const int buf = i & 1, use = i >> 1;
      const int m0 = mt * 256 + rank * kTileRows + quarter * 32, n0 = nt * kPairN;
      tc::named_bar_sync(1, 32 * kOutWarps);  // the last tile's scales are read
      {
        static_assert(kPairN == 32 * kOutWarps, "one channel per epilogue thread");
        const int n = min(n0 + et, a.N - 1);
        scale[et] = a.ws[n];
        bias[et] = a.bias ? a.bias[n] : 0.f;
      }
      const int m = m0 + lane;
      const float xs = m < a.M ? a.xs[m] : 0.f;
      tc::named_bar_sync(1, 32 * kOutWarps);
      const bool ok = tc::warp_all(!*abort && tc::mbar_wait(&acc_full[buf], use & 1, abort));
      tc::tc_fence_after();
      const int rows = min(32, a.M - m0);
#pragma unroll 1
      for (int c = half * (kPairN / 2); c < (half + 1) * (kPairN / 2); c += kCols) {
        float v[kCols];
#pragma unroll
        for (int h = 0; h < kCols; h += 32)
          tc::tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + buf * kPairN + c + h, *reinterpret_cast<float(*)[32]>(&v[h]));
        tc::tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < kCols; j += 4) {
          const float4 s = *reinterpret_cast<const float4 *>(&scale[c + j]);
          const float4 b = *reinterpret_cast<const float4 *>(&bias[c + j]);
          v[j] = fmaf((float)__float_as_int(v[j]) * xs, s.x, b.x);
          v[j + 1] = fmaf((float)__float_as_int(v[j + 1]) * xs, s.y, b.y);
          v[j + 2] = fmaf((float)__float_as_int(v[j + 2]) * xs, s.z, b.z);
          v[j + 3] = fmaf((float)__float_as_int(v[j + 3]) * xs, s.w, b.w);
        }
        if (!ok) {
#pragma unroll
          for (int j = 0; j < kCols; ++j) v[j] = NAN;
        }
        // a row of 128 output bytes per lane, its 16-byte chunks swizzled by the row
        constexpr int kPer = 16 / (int)sizeof(T);  // values per 16-byte chunk
#pragma unroll
        for (int j = 0; j < kCols; j += kPer) {
          const uint32_t at = stage + lane * 128 + (((j / kPer) ^ (lane & 7)) << 4);
          if constexpr (sizeof(T) == 2)
            tc::st_shared_v4(at, tc::pack_bf16(v[j], v[j + 1]), tc::pack_bf16(v[j + 2], v[j + 3]),
                             tc::pack_bf16(v[j + 4], v[j + 5]), tc::pack_bf16(v[j + 6], v[j + 7]));
          else
            tc::st_shared_f4(at, make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
        }
        __syncwarp();
        T *y = static_cast<T *>(a.y) + (long long)m0 * a.N + n0 + c;
        if (a.vec_ok) {  // four rows of 128 bytes per store
          const int chunk = lane & 7, col = chunk * (16 / (int)sizeof(T));
          if (n0 + c + col < a.N) {
#pragma unroll
            for (int r = lane >> 3; r < 32; r += 4) {
              const float4 w = tc::ld_shared_f4(stage + r * 128 + ((chunk ^ (r & 7)) << 4));
              if (r < rows) *reinterpret_cast<float4 *>(y + (long long)r * a.N + col) = w;
            }
          }
        } else {
          for (int r = 0; r < rows; ++r)
#pragma unroll
            for (int col = lane; col < kCols; col += 32) {
              const uint32_t byte = col * (int)sizeof(T);
              const uint32_t at = stage + r * 128 + (((byte >> 4) ^ (r & 7)) << 4) + (byte & 15);
              if constexpr (sizeof(T) == 2) {
                uint16_t w;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(at));
                if (n0 + c + col < a.N) reinterpret_cast<uint16_t *>(y)[(long long)r * a.N + col] = w;
              } else {
                uint32_t w;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(at));
                if (n0 + c + col < a.N) reinterpret_cast<uint32_t *>(y)[(long long)r * a.N + col] = w;
              }
            }
        }
        __syncwarp();
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        arrive_cluster(map_rank(tc::smem_u32(&acc_empty[buf]), 0));
        if (!ok) atomicExch(&g_timeout, 1);
      }
    }
  }
  if (lane == 0 && *abort)
    for (int r = 0; r < 2; ++r) st_cluster_i(map_rank(tc::smem_u32(&sm.gave_up), r), 1);
  __syncwarp();
  cluster_sync();  // the pair's products are done on both sides, and its copies if no wait gave up
  if (sm.gave_up) {
    // Both CTAs' copies must have landed before either leaves.  The leader's barriers count both, so
    // the one that has asked for fewer stages first asks for those that the other has asked for:
    // they are free, since the other one's wait for them ended (their contents are not used).
    if (threadIdx.x == 0) {
      const int mine = sm.filled, wanted = max(mine, ld_cluster_i(map_rank(tc::smem_u32(&sm.filled), rank ^ 1)));
      const uint32_t leader_full = map_rank(tc::smem_u32(&full[0]), 0);
      for (int k = mine; k < wanted; ++k) {
        const int st = k % kPairStages;
        const uint32_t sa = tc::smem_u32(ring) + st * kPairStageBytes;
        if (rank == 0) tc::mbar_arrive_expect_tx(&full[st], 2 * kPairStageBytes);
        tma_load_pair(sa, &mx, leader_full + st * 8, 0, 0);
        tma_load_pair(sa + kTileBytes, &mw, leader_full + st * 8, 0, 0);
      }
      if (rank == 0)
        for (int k = max(wanted - kPairStages, 0); k < wanted; ++k)
          tc::mbar_wait_drain(&full[k % kPairStages], (k / kPairStages) & 1);
    }
    __syncwarp();
    cluster_sync();
  }
  if (warp == 1) {
    tc::tc_fence_after();
    tmem_dealloc_pair(tmem, 2 * kPairN);
  }
}

// ------------------------------------------------------------------ host side
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

int sm_count() {
  static std::atomic<int> cached[kMaxDevices];
  int dev = 0, v = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 148;
  v = cached[dev].load();
  if (!v) {
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) v = 148;
    cached[dev].store(v);
  }
  return v;
}

template <typename T, int BT>
int launch_split(const CUtensorMap &mx, const CUtensorMap &mw, const Args &a, cudaStream_t s) {
  static std::atomic<bool> set[kMaxDevices];
  cudaError_t e = allow_smem(split_kernel<T, BT>, Split<BT>::kBytes, set);
  if (e != cudaSuccess) return cuda_err("int8_linear", e);
  const int n_tiles = (a.N + kTileRows - 1) / kTileRows, m_tiles = (a.M + BT - 1) / BT;
  // Split K while each CTA keeps two K steps and the CTAs fit on the SMs at once: two per SM up
  // to 64 tokens (64 x 16384 x 2048: 11.4 us with 256 CTAs, 12.8 with 128), one with 128, whose
  // sums to exchange cost more than more CTAs gain (777 x 1001 x 2050: 10.6 us with one per SM,
  // 16.4 with two; 128 x 2048 x 2048: 7.1 us split four ways, 11.8 eight).
  const int room = sm_count() * (BT <= 64 ? 2 : 1);
  int S = 1;
  constexpr int kMost = BT <= 64 ? kMaxSplit : kMaxSplit / 2;
  while (S < kMost && 2LL * S * n_tiles * m_tiles <= room && a.k_steps >= 4 * S) S *= 2;
  e = race::launch_early(split_kernel<T, BT>, dim3((unsigned)(n_tiles * S), (unsigned)m_tiles), dim3(kThreads),
                         Split<BT>::kBytes, s, (unsigned)S, mx, mw, a, S);
  if (e != cudaSuccess) return cuda_err("int8_linear", e);
  return race::launched("int8_linear");
}

template <typename T>
int launch_pair(const CUtensorMap &mx, const CUtensorMap &mw, const Args &a, cudaStream_t s) {
  static std::atomic<bool> set[kMaxDevices];
  const cudaError_t e = allow_smem(pair_kernel<T>, sizeof(PairSmem), set);
  if (e != cudaSuccess) return cuda_err("int8_linear", e);
  const long long tiles = (long long)a.m_tiles * a.n_tiles, pairs = sm_count() / 2;
  pair_kernel<T><<<(unsigned)(2 * (tiles < pairs ? tiles : pairs)), kPairThreads, sizeof(PairSmem), s>>>(mx, mw, a);
  return race::launched("int8_linear");
}

template <typename T>
int launch(const int8_t *xq, int64_t x_stride, const int8_t *wq, int64_t w_stride, int64_t K, Args a, cudaStream_t s) {
  a.m_tiles = (a.M + 255) / 256;
  a.n_tiles = (a.N + kPairN - 1) / kPairN;
  // The pair kernel once its tiles occupy a third of the pairs (1024 x 2048 x 2048, 32 tiles: 11.7
  // us against 13.8 split; 777 x 1001 x 2050, 16 tiles: 14.9 against 10.6; 1024 x 1024 x 2048, 16
  // tiles: 10.8 against 9.2).
  const bool pairs = a.M > 128 && (long long)a.m_tiles * a.n_tiles >= sm_count() / 6;
  const int BT = pairs ? 128 : a.M <= 16 ? 16 : a.M <= 32 ? 32 : a.M <= 64 ? 64 : 128;
  CUtensorMap mx, mw;
  if (!race::bind_context() || !race::make_byte_rows_map(&mx, xq, a.M, K, x_stride, BT) || !race::make_byte_rows_map(&mw, wq, a.N, K, w_stride, kTileRows))
    return err(RACE_ERR_CUDA, "race_int8_linear: no tensor map for M=%lld, N=%lld", a.M, a.N);
  if (pairs) return launch_pair<T>(mx, mw, a, s);
  switch (BT) {
    case 16: return launch_split<T, 16>(mx, mw, a, s);
    case 32: return launch_split<T, 32>(mx, mw, a, s);
    case 64: return launch_split<T, 64>(mx, mw, a, s);
    default: return launch_split<T, 128>(mx, mw, a, s);
  }
}

// race_set_status_check(1): wait for the stream and report a wait that gave up (a captured call
// does not run now, so there is nothing to wait for).
int check_status(cudaStream_t s) {
  if (!race::status_check_on()) return RACE_OK;
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  cudaError_t e = cudaStreamIsCapturing(s, &capture);
  if (e != cudaSuccess) return cuda_err("int8_linear", e);
  if (capture != cudaStreamCaptureStatusNone) return RACE_OK;
  int flag = 0;
  e = cudaStreamSynchronize(s);
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
  // tile coordinates and the number of 128 x 128 tiles (times a split of 8) are 32-bit; a
  // grid's second dimension holds the token tiles
  if (M < 1 || N < 1 || M > (1 << 23) - 128 || N > (1 << 27) || ((M + 127) / 128) * ((N + 127) / 128) > (1 << 27))
    return err(RACE_ERR_SHAPE, "race_int8_linear: M=%lld or N=%lld out of range", M, N);
  if (K < 1 || K > kMaxK) return err(RACE_ERR_SHAPE, "race_int8_linear: K=%lld not in 1..%lld", K, kMaxK);
  if (x_stride < K || w_stride < K) return err(RACE_ERR_SHAPE, "race_int8_linear: row stride below K=%lld", K);
  if (((reinterpret_cast<uintptr_t>(xq) | reinterpret_cast<uintptr_t>(wq) | (uintptr_t)x_stride | (uintptr_t)w_stride) & 15) ||
      ((reinterpret_cast<uintptr_t>(x_scale) | reinterpret_cast<uintptr_t>(w_scale) | reinterpret_cast<uintptr_t>(bias)) & 3))
    return err(RACE_ERR_ALIGN, "race_int8_linear: 8-bit rows must start at multiples of 16 bytes");
  const int size = race::value_size(dtype);
  if (const int rc = race::check_values("race_int8_linear", {{y, size}})) return rc;
  Args a{x_scale, w_scale, bias, y, (int)M, (int)N, (int)((K + kBK - 1) / kBK), 0, 0,
         (N * size) % 16 == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0, race::withhold_first_load() ? 1 : 0,
         race::current_wait_limit()};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int rc = dtype == RACE_BF16 ? launch<__nv_bfloat16>(xq, x_stride, wq, w_stride, K, a, s)
                                    : launch<float>(xq, x_stride, wq, w_stride, K, a, s);
  return rc == RACE_OK ? check_status(s) : rc;
}

}  // extern "C"
