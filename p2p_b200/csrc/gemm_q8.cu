// gemm_q8.cu -- products of 8-bit integer rows with a scale each: a projection (bias, residual), or the
// gate and up projections of a feed-forward block with their activation and product (SILU_MUL,
// src/scripts/lfm-engine/kernels.js:321-339).
//
// Sums are whole numbers in 32 bits on tcgen05.mma.kind::i8, so every split of them gives the same
// result; the scales, the activation and what is added follow in f32.  Two kernels:
//   wide_kernel    many tokens: a cluster of two CTAs per 256-token tile and one
//                  tcgen05.mma.cta_group::2 stream, persistent;
//   narrow_kernel  few tokens, bound by the weights' bytes: the weights are the MMA's 128 rows and the
//                  tokens its columns, k split over a cluster whose CTAs add their sums through
//                  distributed shared memory.
// Every mbarrier wait is bounded (about one second): a wait that gives up sets the device error word,
// every role of the CTA stops, the copies and MMAs in flight are waited for, the TMEM is freed and the
// CTA returns.
#include <cuda.h>

#include <algorithm>
#include <climits>

#include "common.cuh"
#include "gemm_common.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace p2p {
namespace {

using namespace sm100;

constexpr int kStep = 128;  // codes of k per stage: one 128-byte swizzled row per operand row

struct Q8Params {
  int32_t m, n, k;
  int32_t act;
  const float* xs;
  const float* ws;
  const float* us;    // gate form: the up rows' scales
  const float* bias;
  const void* res;
  void* y;
  int64_t ld_res, ld_y;
  int32_t* err;
  // wide_kernel
  int32_t tiles_n, whole, items;  // tiles along n; tiles of full width; work items in all
  int32_t wide;                   // y and res rows on 16-byte boundaries
  // narrow_kernel
  int32_t tokens;     // columns of a tile
  int32_t stages;
};

// act(g) * u.  The exponential and the quotient are approximations of 2 units in the last place each.
__device__ __forceinline__ float act_mul(float g, float u, int act) {
  const float t = act == kActSilu ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
  return __fdividef(g, 1.f + __expf(-t)) * u;
}

__device__ __forceinline__ float scaled(uint32_t acc, float xs, float ws) {
  return __fmul_rn(__fmul_rn(float(int(acc)), xs), ws);
}

// ---- many tokens ------------------------------------------------------------------------------------
constexpr int kRows = 128;      // token rows of a CTA (256 of a pair)
constexpr int kWidth = 256;     // columns of a whole tile; the last tiles may be halved
constexpr int kEpiWarps = 8;
constexpr int kTmaWarp = kEpiWarps, kMmaWarp = kEpiWarps + 1;
constexpr int kWideThreads = 32 * (kEpiWarps + 2);
constexpr int kBoxRows = 64;    // weight rows per TMA box
constexpr uint32_t kTileBytes = kRows * kStep;          // x, and a CTA's half of the weights
constexpr int kWideStages = 5;
constexpr int kPitch = 33;

struct __align__(1024) WideSmem {
  uint8_t a[kWideStages][kTileBytes];
  uint8_t b[kWideStages][kTileBytes];
  float turn[kEpiWarps][32 * kPitch];   // a warp's 32 x 32 outputs, to store rows along lanes
  float col[kEpiWarps][2][128];         // a warp's columns: scales, and biases or the up scales
  uint64_t full[kWideStages], empty[kWideStages];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t mma_done;
  uint32_t tmem_base;
  volatile int abort_flag;
};

struct Item {
  int m0, n0, bn;  // first token and column, columns of the MMA
};
// Tiles in order of rows, then columns; tiles from `whole` on as two halves.  GATE: a tile of bn MMA
// columns covers bn / 2 columns of h.
template <bool GATE>
__device__ __forceinline__ Item item_of(const Q8Params& p, int i) {
  constexpr int kCols = GATE ? kWidth / 2 : kWidth;
  Item it;
  const int t = i < p.whole ? i : p.whole + (i - p.whole) / 2;
  it.m0 = t / p.tiles_n * (2 * kRows);
  it.n0 = t % p.tiles_n * kCols;
  it.bn = kWidth;
  if (i >= p.whole) {
    it.n0 += ((i - p.whole) & 1) * (kCols / 2);
    it.bn = kWidth / 2;
  } else if (p.n - it.n0 <= kCols / 2) {
    it.bn = kWidth / 2;
  }
  return it;
}

// 32 consecutive columns of 32 rows (a row per lane), from n on.
template <class T>
__device__ __forceinline__ void store_block(const Q8Params& p, float (&v)[32], int m_base, int lane,
                                            int n, float* turn) {
  const int m = m_base + lane;
  if (p.wide && n + 32 <= p.n) {
    if (m >= p.m) return;
    constexpr int V = 16 / sizeof(T);
    union {
      uint4 u;
      T e[V];
    } w;
    if (p.res) {
      const uint4* r = reinterpret_cast<const uint4*>(static_cast<const T*>(p.res) +
                                                      int64_t(m) * p.ld_res + n);
#pragma unroll
      for (int i = 0; i < 32 / V; ++i) {
        w.u = r[i];
#pragma unroll
        for (int j = 0; j < V; ++j) v[i * V + j] = __fadd_rn(v[i * V + j], to_f32(w.e[j]));
      }
    }
    uint4* d = reinterpret_cast<uint4*>(static_cast<T*>(p.y) + int64_t(m) * p.ld_y + n);
#pragma unroll
    for (int i = 0; i < 32 / V; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) w.e[j] = from_f32<T>(v[i * V + j]);
      d[i] = w.u;
    }
    return;
  }
  // rows that start anywhere, or end inside the block: a row at a time along the lanes
#pragma unroll
  for (int c = 0; c < 32; ++c) turn[lane * kPitch + c] = v[c];
  __syncwarp();
  const int rows = min(32, p.m - m_base), c = n + lane;
  if (c < p.n) {
    T* d = static_cast<T*>(p.y) + int64_t(m_base) * p.ld_y + c;
    const T* r = static_cast<const T*>(p.res) + int64_t(m_base) * p.ld_res + c;
#pragma unroll 4
    for (int i = 0; i < rows; ++i) {
      float y = turn[i * kPitch + lane];
      if (p.res) y = __fadd_rn(y, to_f32(r[int64_t(i) * p.ld_res]));
      d[int64_t(i) * p.ld_y] = from_f32<T>(y);
    }
  }
  __syncwarp();
}

// The epilogue of one item by epilogue warp `warp`: TMEM lane quarter warp & 3, every other block of 32
// columns.
template <class T, bool GATE, class Release>
__device__ __forceinline__ void wide_epilogue(const Q8Params& p, WideSmem& s, uint32_t acc,
                                              const Item& it, int m0, int warp, int lane,
                                              Release release) {
  const int quarter = warp & 3, half = warp >> 2;
  const int cols = GATE ? it.bn / 2 : it.bn, blocks = cols / 32;
  const uint32_t at = acc + (uint32_t(quarter * 32) << 16);
  const int m_base = m0 + quarter * 32;
  float* ws = s.col[warp][0];
  float* second = s.col[warp][1];
  const float xs = m_base + lane < p.m ? p.xs[m_base + lane] : 0.f;
  for (int b = half, i = lane; b < blocks; b += 2, i += 32) {
    const int c = it.n0 + b * 32 + lane;
    ws[i] = c < p.n ? p.ws[c] : 0.f;
    if constexpr (GATE) second[i] = c < p.n ? p.us[c] : 0.f;
    else if (p.bias) second[i] = c < p.n ? p.bias[c] : 0.f;
  }
  __syncwarp();
  for (int b = half, i = 0; b < blocks; b += 2, i += 32) {
    uint32_t r[32];
    float v[32];
    tmem_ld32(at + b * 32, r);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = scaled(r[j], xs, ws[i + j]);
    if constexpr (GATE) {
      tmem_ld32(at + cols + b * 32, r);
      tmem_ld_wait();
      if (p.act == kActSilu) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          v[j] = act_mul(v[j], scaled(r[j], xs, second[i + j]), kActSilu);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          v[j] = act_mul(v[j], scaled(r[j], xs, second[i + j]), kActGelu);
      }
    } else if (p.bias) {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = __fadd_rn(v[j], second[i + j]);
    }
    if (b + 2 >= blocks) {  // everything of this warp is in registers
      tc_fence_before();
      __syncwarp();
      release();
    }
    if (m_base < p.m && it.n0 + b * 32 < p.n)
      store_block<T>(p, v, m_base, lane, it.n0 + b * 32, s.turn[warp]);
    __syncwarp();
  }
}

// A cluster of two CTAs per tile of 256 tokens.  The even CTA (rank 0) issues the MMAs of both; each
// CTA's TMA loads its own 128 token rows and its half of the tile's weight rows (GATE: rank 0 the gate's,
// rank 1 the up's) into its own shared memory, all completing on the even CTA's ring barriers; commits
// arrive on both CTAs' barriers.
template <class T, bool GATE>
__global__ void __launch_bounds__(kWideThreads, 1)
    wide_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                const __grid_constant__ CUtensorMap tm_u, const __grid_constant__ Q8Params p) {
  extern __shared__ uint8_t smem_raw[];
  WideSmem& s = *reinterpret_cast<WideSmem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = int(cluster_id_x()), pairs = int(cluster_count_x());
  const int nk = (p.k + kStep - 1) / kStep;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kWideStages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.acc_full[i], 1);
      mbar_init(&s.acc_empty[i], 2 * kEpiWarps);
    }
    mbar_init(&s.mma_done, 1);
    s.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) tmem_alloc_pair(&s.tmem_base, 512);
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers initialised and visible, the pair's TMEM allocated
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  grid_dependency_wait();
  launch_dependents();

  if (warp == kTmaWarp) {
    if (lane == 0) {
      const CUtensorMap* tm_b = GATE && rank ? &tm_u : &tm_w;
      prefetch_tensormap(&tm_x);
      prefetch_tensormap(tm_b);
      uint32_t g = 0;  // ring slot counter, continuous across items
      bool ok = true;
      for (int i = pair; i < p.items && ok; i += pairs) {
        const Item it = item_of<GATE>(p, i);
        const int m0 = it.m0 + int(rank) * kRows, half = it.bn / 2;
        const int n0 = GATE ? it.n0 : it.n0 + int(rank) * half;
        for (int kt = 0; kt < nk; ++kt, ++g) {
          const uint32_t st = g % kWideStages;
          if (g >= kWideStages &&
              !gemm_wait(s.abort_flag, &s.empty[st], ((g / kWideStages) - 1) & 1, p.err)) {
            ok = false;
            break;
          }
          const uint32_t full0 = cluster_map(smem_u32(&s.full[st]), 0);
          if (rank == 0) mbar_arrive_expect_tx(&s.full[st], 2 * (kTileBytes + half * kStep));
          tma_load_2d_pair(s.a[st], &tm_x, kt * kStep, m0, full0);
          for (int r = 0; r < half; r += kBoxRows)
            tma_load_2d_pair(s.b[st] + r * kStep, tm_b, kt * kStep, n0 + r, full0);
        }
      }
      if (!ok) {  // let the copies already in flight land before the CTA exits
        if (rank == 0) {
          for (uint32_t h = g > kWideStages ? g - kWideStages : 0; h < g; ++h) {
            const uint64_t t0 = globaltimer_ns();
            while (!mbar_try_wait(&s.full[h % kWideStages], (h / kWideStages) & 1) &&
                   globaltimer_ns() - t0 < kGemmWaitNs) {
            }
          }
        } else {  // its loads complete on the even CTA's barriers: give them time to land
          const uint64_t t0 = globaltimer_ns();
          while (globaltimer_ns() - t0 < 100000) {
          }
        }
      }
    }
  } else if (warp == kMmaWarp) {
    if (rank == 0) {
      const uint64_t adesc0 = smem_desc_sw128(smem_u32(s.a[0]), 16, 1024);
      const uint64_t bdesc0 = smem_desc_sw128(smem_u32(s.b[0]), 16, 1024);
      bool ok = true, issued = false;
      uint32_t g = 0;
      int n = 0;  // items of this pair
      for (int i = pair; i < p.items && ok; i += pairs, ++n) {
        const int b = n & 1, u = n >> 1;  // accumulator buffer, its use count
        if (u > 0 &&
            !(ok = gemm_wait_warp(s.abort_flag, &s.acc_empty[b], (u - 1) & 1, p.err, lane)))
          break;
        tc_fence_after();
        const uint32_t idesc = idesc_i8(2 * kRows, item_of<GATE>(p, i).bn);
        const uint32_t acc = tmem + uint32_t(b * kWidth);
        for (int kt = 0; kt < nk; ++kt, ++g) {
          const uint32_t st = g % kWideStages;
          if (!(ok = gemm_wait_warp(s.abort_flag, &s.full[st], (g / kWideStages) & 1, p.err, lane)))
            break;
          tc_fence_after();
          if (elect_one()) {
            // a step of 32 codes is +32 bytes (2 address units) inside the 128-byte swizzled rows
            const uint64_t ad = adesc0 + uint64_t(st) * (kTileBytes >> 4),
                           bd = bdesc0 + uint64_t(st) * (kTileBytes >> 4);
#pragma unroll
            for (int kk = 0; kk < kStep / 32; ++kk)
              mma_pair_i8_ss(acc, ad + 2 * kk, bd + 2 * kk, idesc, (kt > 0 || kk > 0) ? 1u : 0u);
            mma_pair_commit(&s.empty[st], 0x3);
          }
          issued = true;
          __syncwarp();
        }
        if (ok && elect_one()) mma_pair_commit(&s.acc_full[b], 0x3);
        __syncwarp();
      }
      if (issued) {  // no MMA of the pair may still run when the TMEM is freed
        if (elect_one()) mma_pair_commit(&s.mma_done, 0x1);
        __syncwarp();
        if (lane == 0) {
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(&s.mma_done, 0) && globaltimer_ns() - t0 < kGemmWaitNs) {
          }
        }
        __syncwarp();
      }
    }
  } else {
    int n = 0;
    for (int i = pair; i < p.items; i += pairs, ++n) {
      const int b = n & 1, u = n >> 1;
      __syncwarp();
      if (!gemm_wait_warp(s.abort_flag, &s.acc_full[b], u & 1, p.err, lane)) break;
      tc_fence_after();
      const uint32_t empty0 = cluster_map(smem_u32(&s.acc_empty[b]), 0);
      const Item it = item_of<GATE>(p, i);
      wide_epilogue<T, GATE>(p, s, tmem + uint32_t(b * kWidth), it, it.m0 + int(rank) * kRows, warp,
                             lane, [&] {
                               if (lane == 0) mbar_arrive_cluster(empty0);
                             });
    }
  }

  tc_fence_before();
  cluster_sync();  // neither CTA leaves while the other may still reach into it
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---- few tokens -------------------------------------------------------------------------------------
// A tile: 128 weight rows (GATE: 64 gate rows above 64 up rows) x up to kMostTokens tokens, its k in the
// hands of the CTAs of one cluster.  Every CTA sums its part of k in TMEM and hands the sums, by token, to
// the CTA that finishes that token; each CTA adds what it was handed and stores.
constexpr int kNarrowThreads = 256;
constexpr int kMostTokens = 128;
constexpr int kMostSplit = 8;
constexpr int kMostStages = 12;

struct NarrowHead {  // in front of the ring and the sums
  uint64_t full[kMostStages], empty[kMostStages];
  uint64_t done;
  uint32_t tmem_base;
  volatile int abort_flag;
};
static_assert(sizeof(NarrowHead) <= 1024, "the head is one swizzle atom");

__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

template <class T, bool GATE>
__global__ void __launch_bounds__(kNarrowThreads)
    narrow_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                  const __grid_constant__ CUtensorMap tm_u, const __grid_constant__ Q8Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  NarrowHead& s = *reinterpret_cast<NarrowHead*>(base);
  uint8_t* ring = base + 1024;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = int(cluster_ctas()), rank = int(cluster_ctarank());
  const uint32_t stage_bytes = kTileBytes + uint32_t(p.tokens) * kStep;
  uint32_t* sums = reinterpret_cast<uint32_t*>(ring + p.stages * stage_bytes);  // [split][own][128]
  const int own = (p.tokens + split - 1) / split;
  const int tile = blockIdx.x / split;
  constexpr int kCols = GATE ? 64 : 128;
  const int n0 = tile % p.tiles_n * kCols, m0 = tile / p.tiles_n * p.tokens;
  const int nk = (p.k + kStep - 1) / kStep;
  const int k0 = int(int64_t(nk) * rank / split), k1 = int(int64_t(nk) * (rank + 1) / split);
  const uint32_t tmem_cols = p.tokens <= 32 ? 32 : p.tokens <= 64 ? 64 : 128;
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    mbar_init(&s.done, 1);
    s.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(&s.tmem_base, tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  // another CTA's shared memory is not touched before that CTA runs
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  grid_dependency_wait();
  launch_dependents();

  if (warp == 0) {
    if (lane == 0) {
      uint32_t g = 0;
      bool ok = true;
      for (int kt = k0; kt < k1; ++kt, ++g) {
        const uint32_t st = g % p.stages;
        if (g >= uint32_t(p.stages) &&
            !gemm_wait(s.abort_flag, &s.empty[st], ((g / p.stages) - 1) & 1, p.err)) {
          ok = false;
          break;
        }
        uint8_t* a = ring + st * stage_bytes;
        mbar_arrive_expect_tx(&s.full[st], stage_bytes);
        tma_load_2d(a, &tm_w, kt * kStep, n0, &s.full[st]);
        if constexpr (GATE) tma_load_2d(a + kTileBytes / 2, &tm_u, kt * kStep, n0, &s.full[st]);
        else tma_load_2d(a + kTileBytes / 2, &tm_w, kt * kStep, n0 + 64, &s.full[st]);
        tma_load_2d(a + kTileBytes, &tm_x, kt * kStep, m0, &s.full[st]);
      }
      if (!ok) {  // let the copies already in flight land before the CTA exits
        for (uint32_t h = g > uint32_t(p.stages) ? g - p.stages : 0; h < g; ++h) {
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(&s.full[h % p.stages], (h / p.stages) & 1) &&
                 globaltimer_ns() - t0 < kGemmWaitNs) {
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t idesc = idesc_i8(128, p.tokens);
    const uint64_t adesc0 = smem_desc_sw128(smem_u32(ring), 16, 1024);
    bool ok = true;
    uint32_t g = 0;
    for (int kt = k0; kt < k1; ++kt, ++g) {
      const uint32_t st = g % p.stages;
      if (!(ok = gemm_wait_warp(s.abort_flag, &s.full[st], (g / p.stages) & 1, p.err, lane))) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t ad = adesc0 + uint64_t(st) * (stage_bytes >> 4), bd = ad + (kTileBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < kStep / 32; ++kk)
          mma_i8_ss(tmem, ad + 2 * kk, bd + 2 * kk, idesc, (g > 0 || kk > 0) ? 1u : 0u);
        mma_commit(&s.empty[st]);
      }
      __syncwarp();
    }
    // also where a wait gave up: no MMA may still run when the TMEM is freed
    if (elect_one()) mma_commit(&s.done);
    __syncwarp();
    if (!ok && lane == 0) {
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(&s.done, 0) && globaltimer_ns() - t0 < kGemmWaitNs) {
      }
    }
    __syncwarp();
  }

  // the sums, token by token, to the CTAs that finish them
  bool ok = true;
  if (warp >= 4) ok = gemm_wait_warp(s.abort_flag, &s.done, 0, p.err, lane);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (warp >= 4 && ok) {
    tc_fence_after();
    const uint32_t at = tmem + (uint32_t((warp & 3) * 32) << 16);
    const int ch = (warp & 3) * 32 + lane;
    for (int t0 = 0; t0 < p.tokens; t0 += 8) {
      uint32_t r[8];
      tmem_ld8(at + t0, r);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int t = t0 + j, to = t / own;
        st_cluster(cluster_map(smem_u32(sums + (rank * own + t - to * own) * 128 + ch), to), r[j]);
      }
    }
  }
  if (s.abort_flag && lane == 0)  // nothing of a sum that lacks a part is stored
    for (int i = 0; i < split; ++i)
      st_cluster(cluster_map(smem_u32(const_cast<int*>(&s.abort_flag)), i), 1u);
  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
  if (s.abort_flag) return;

  for (int i = threadIdx.x; i < own * kCols; i += kNarrowThreads) {
    const int c = i % kCols, tl = i / kCols, t = rank * own + tl;
    const int m = m0 + t, n = n0 + c;
    if (t >= p.tokens || m >= p.m || n >= p.n) continue;
    int acc = 0, acc2 = 0;
    for (int j = 0; j < split; ++j) {
      acc += int(sums[(j * own + tl) * 128 + c]);
      if constexpr (GATE) acc2 += int(sums[(j * own + tl) * 128 + 64 + c]);
    }
    const float xs = p.xs[m];
    float y = scaled(uint32_t(acc), xs, p.ws[n]);
    if constexpr (GATE) {
      y = act_mul(y, scaled(uint32_t(acc2), xs, p.us[n]), p.act);
    } else {
      if (p.bias) y = __fadd_rn(y, p.bias[n]);
      if (p.res)
        y = __fadd_rn(y, to_f32(static_cast<const T*>(p.res)[int64_t(m) * p.ld_res + n]));
    }
    static_cast<T*>(p.y)[int64_t(m) * p.ld_y + n] = from_f32<T>(y);
  }
}

// ---- host -------------------------------------------------------------------------------------------
// Rows of codes in boxes of 128 codes x box_rows, 128-byte swizzle; what lies outside reads as 0.
bool map_codes(CUtensorMap* m, const Q8Rows& r, uint32_t box_rows) {
  auto enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[2] = {cuuint64_t(r.cols), cuuint64_t(r.rows)};
  cuuint64_t strides[1] = {cuuint64_t(r.ld)};
  cuuint32_t box[2] = {kStep, box_rows};
  cuuint32_t estr[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, r.q, dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t launch_cluster(const void* fn, int64_t ctas, int threads, size_t smem, int cluster,
                           void** args, cudaStream_t stream) {
  if (ctas > INT32_MAX) return cudaErrorInvalidValue;
  cudaLaunchAttribute at[2] = {};
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = unsigned(cluster);
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelExC(&cfg, fn, args);
}

template <class T, bool GATE>
cudaError_t launch_wide(Q8Params p, const GemmQ8Args& a, int num_sms, cudaStream_t stream) {
  CUtensorMap tx, tw, tu;
  if (!map_codes(&tx, a.x, kRows) || !map_codes(&tw, a.w, kBoxRows) ||
      !map_codes(&tu, GATE ? a.up : a.w, kBoxRows))
    return cudaErrorInvalidValue;
  const void* fn = reinterpret_cast<const void*>(&wide_kernel<T, GATE>);
  const size_t smem = sizeof(WideSmem) + 1024;
  static PerDeviceOnce setup;
  int max_pairs = 0;
  cudaError_t e = per_device_once(setup, [&](int& pairs) {
    cudaError_t err =
        cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (err != cudaSuccess) return err;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 2;
    at.val.clusterDim.y = 1;
    at.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2);
    cfg.blockDim = dim3(kWideThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaOccupancyMaxActiveClusters(&pairs, fn, &cfg);
  }, &max_pairs);
  if (e != cudaSuccess) return e;
  if (max_pairs <= 0) return cudaErrorInvalidConfiguration;
  constexpr int kCols = GATE ? kWidth / 2 : kWidth;
  const int64_t tiles_n = (int64_t(p.n) + kCols - 1) / kCols;
  const int64_t tiles = tiles_n * ((int64_t(p.m) + 2 * kRows - 1) / (2 * kRows));
  if (2 * tiles > INT32_MAX) return cudaErrorInvalidValue;
  // the last wave's tiles are halved where their halves still fit one wave
  const int64_t rest = tiles % max_pairs;
  p.tiles_n = int32_t(tiles_n);
  p.whole = int32_t(2 * rest <= max_pairs ? tiles - rest : tiles);
  p.items = int32_t(p.whole + 2 * (tiles - p.whole));
  void* args[] = {&tx, &tw, &tu, &p};
  return launch_cluster(fn, 2 * std::min<int64_t>(p.items, max_pairs), kWideThreads, smem, 2, args,
                        stream);
}

template <class T, bool GATE>
cudaError_t launch_narrow(Q8Params p, const GemmQ8Args& a, int num_sms, cudaStream_t stream) {
  // columns of an MMA: 8, 16, 24, or multiples of 16
  const int tokens = std::min(kMostTokens, p.m <= 24 ? (p.m + 7) / 8 * 8 : (p.m + 15) / 16 * 16);
  CUtensorMap tx, tw, tu;
  if (!map_codes(&tx, a.x, unsigned(tokens)) || !map_codes(&tw, a.w, 64) ||
      !map_codes(&tu, GATE ? a.up : a.w, 64))
    return cudaErrorInvalidValue;
  constexpr int kCols = GATE ? 64 : 128;
  const int64_t tiles_n = (int64_t(p.n) + kCols - 1) / kCols;
  const int64_t tiles = tiles_n * ((int64_t(p.m) + tokens - 1) / tokens);
  const int nk = (p.k + kStep - 1) / kStep;
  int split = 1;
  while (2 * split <= std::min(kMostSplit, nk) && tiles * 2 * split <= 2 * num_sms) split *= 2;
  const int own = (tokens + split - 1) / split;
  const int stage = int(kTileBytes) + tokens * kStep, sums = split * own * 128 * 4;
  const int room = (tokens <= 64 ? 113 : 226) * 1024 - 2048 - sums;
  const int steps = (nk + split - 1) / split;
  p.stages = std::max(1, std::min({kMostStages, steps, room / stage}));
  p.tokens = tokens;
  p.tiles_n = int32_t(tiles_n);
  const size_t smem = 2048 + size_t(p.stages) * stage + sums;
  const void* fn = reinterpret_cast<const void*>(&narrow_kernel<T, GATE>);
  static PerDeviceOnce attrs;
  cudaError_t e = per_device_once(attrs, [&](int&) {
    return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
  });
  if (e != cudaSuccess) return e;
  void* args[] = {&tx, &tw, &tu, &p};
  return launch_cluster(fn, tiles * split, kNarrowThreads, smem, split, args, stream);
}

bool on16(const void* p, int64_t pitch_bytes) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && pitch_bytes % 16 == 0;
}

template <class T, bool GATE>
cudaError_t launch_q8(const Q8Params& p, const GemmQ8Args& a, int num_sms, cudaStream_t s) {
  return p.m <= kMostTokens ? launch_narrow<T, GATE>(p, a, num_sms, s)
                            : launch_wide<T, GATE>(p, a, num_sms, s);
}

}  // namespace

cudaError_t launch_gemm_q8(const GemmQ8Args& a, int dtype, int num_sms, cudaStream_t s) {
  Q8Params p{};
  p.m = a.x.rows;
  p.n = a.w.rows;
  p.k = a.x.cols;
  p.act = a.act;
  p.xs = a.x.scale;
  p.ws = a.w.scale;
  p.us = a.up.scale;
  p.bias = a.bias;
  p.res = a.res;
  p.y = a.y;
  p.ld_res = a.ld_res;
  p.ld_y = a.ld_y;
  p.err = a.err;
  const int64_t es = dtype == 0 ? 2 : 4;
  p.wide = on16(a.y, a.ld_y * es) && (!a.res || on16(a.res, a.ld_res * es));
  if (a.up.q) return launch_q8<__half, true>(p, a, num_sms, s);
  return dtype == 0 ? launch_q8<__half, false>(p, a, num_sms, s)
                    : launch_q8<float, false>(p, a, num_sms, s);
}

}  // namespace p2p
