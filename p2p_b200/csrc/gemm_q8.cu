// gemm_q8.cu -- products of 8-bit integer rows with a scale each: a projection (bias, residual), or the
// gate and up projections of a feed-forward block with their activation and product (SILU_MUL,
// src/scripts/lfm-engine/kernels.js:321-339).
//
// Sums are whole numbers in 32 bits on tcgen05.mma.kind::i8, so every split of them gives the same
// result; the scales, the activation and what is added follow in f32.  Two kernels:
//   wide_kernel    many tokens, bound by the MMAs (and, called back to back, by the power limit): a cluster
//                  of two CTAs per 256 x 256 tile and one tcgen05.mma.cta_group::2 stream, persistent, two
//                  accumulators, the last wave's tiles halved.  Gate and up of 4096 tokens (8192 x 2048
//                  each): 76 us alone (3630 TOP/s, 89 % of the tensor pipe's cycles), 86 us among some,
//                  103 us in long runs; 8192 x 2048 x 8192: 81, 88 and 104 us.
//   narrow_kernel  few tokens, bound by the weights' bytes: the weights are the MMA's rows and the tokens
//                  its columns.  The LM head of 32 tokens (65536 x 2048) 24.4 us (5.9 TB/s), gate and up of
//                  one token (2 x 8192 x 2048) 7.0 us, 48 x 2048 x 8192 6.5 us (15 by pairs of CTAs).
// A warp that walks a ring does so as a whole: with its loop in one lane the compiler has to treat what a
// copy takes as different in every lane, and a stage took 200 ns to issue (8192 x 2048 x 8192 98 -> 91 us).
// Every mbarrier wait is bounded (about one second): a wait that gives up sets the device error word,
// every role of the CTA stops, the copies and MMAs in flight are waited for, the TMEM is freed and the
// CTA returns.
#include <cuda.h>

#include <algorithm>
#include <climits>
#include <type_traits>

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
  int32_t wait_deficit;    // bytes more than will arrive that the first stage waits for (a test)
  int32_t tiles_n, items;  // tiles along n; work items in all
  // wide_kernel
  int32_t whole;  // tiles of full width
  int32_t wide;   // y and res rows on 16-byte boundaries
  // narrow_kernel
  int32_t rows, tokens, steps;  // of a tile
  int32_t stages, chunks;       // of the ring; of a stage
  int32_t deep;                 // the tensor maps' third dimension is k in steps of 128
};

// act(g) * u.  The exponential and the reciprocal are approximations of a few units in the last place (the
// f16 of the result has a 2^-11th) that take what is below f32's normal numbers as 0: 1 / (1 + exp(-t)) is
// there from t = -87.3 on, where exp(-t) is still a number, and a large u brings the product back.  So a
// quarter of the sum goes into the reciprocal, and a quarter of that out of it.
template <bool GELU>
__device__ __forceinline__ Pair act_mul(Pair g, Pair u) {
  constexpr float k = GELU ? -1.5957691216057308f * kLog2e : -kLog2e;
  const Pair quarter = pair(0.25f, 0.25f), less = pair(-2.f, -2.f);
  Pair t;
  if constexpr (GELU)
    t = mad2(mul2(g, pair(k, k)), mad2(mul2(g, g), pair(0.044715f, 0.044715f), pair(1.f, 1.f)), less);
  else
    t = mad2(g, pair(k, k), less);
  const Pair d = add2(pair(fast_exp2(t.f[0]), fast_exp2(t.f[1])), quarter);
  Pair r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.f[0]) : "f"(d.f[0]));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.f[1]) : "f"(d.f[1]));
  return mul2(mul2(g, mul2(r, quarter)), u);
}
__device__ __forceinline__ Pair act_mul(Pair g, Pair u, int act) {
  return act == kActSilu ? act_mul<false>(g, u) : act_mul<true>(g, u);
}

__device__ __forceinline__ Pair scaled2(uint32_t a, uint32_t b, Pair xs, Pair ws) {
  return mul2(mul2(pair(float(int(a)), float(int(b))), xs), ws);
}

// ---- many tokens ------------------------------------------------------------------------------------
constexpr int kRows = 128;      // token rows of a CTA (256 of a pair)
constexpr int kWidth = 256;     // columns of a whole tile; the last tiles may be halved
constexpr int kEpiWarps = 8;
constexpr int kTmaWarp = kEpiWarps, kMmaWarp = kEpiWarps + 1;
constexpr int kWideThreads = 32 * (kEpiWarps + 2);
constexpr int kBoxRows = 64;    // weight rows per TMA box
constexpr uint32_t kTileBytes = kRows * kStep;          // x, and a CTA's half of the weights
// A warp's 32 x 32 outputs change hands through shared memory, so that it stores whole stretches of rows:
// 20 words a row of f16, 36 of f32 (both keep 16-byte accesses of a column free of conflicts), and what
// that leaves goes to the ring (8192 x 2048 x 8192 in 84.0 us with 6 stages, 85.0 with 5, 91 with 4).
template <class T>
constexpr int kPitch = sizeof(T) == 4 ? 36 : 20;
template <class T>
constexpr int kWideStages = sizeof(T) == 4 ? 5 : 6;

template <class T>
struct __align__(1024) WideSmem {
  static constexpr int kStages = kWideStages<T>;
  uint8_t a[kStages][kTileBytes];
  uint8_t b[kStages][kTileBytes];
  uint32_t turn[kEpiWarps][32 * kPitch<T>];
  float col[kEpiWarps][2][128];         // a warp's columns: scales, and biases or the up scales
  uint64_t full[kStages], empty[kStages];
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

// 32 consecutive columns, from n on, of 32 rows (a row per lane).  `aligned`: rows on 16-byte boundaries
// that hold all 32 columns, and what is added has been.
template <class T>
__device__ __forceinline__ void store_block(const Q8Params& p, const Pair (&v)[16], int m_base, int lane,
                                            int n, bool aligned, uint32_t* turn) {
  constexpr bool kF16 = sizeof(T) == 2;
  uint4* mine = reinterpret_cast<uint4*>(turn + lane * kPitch<T>);
  // N pairs of this lane's row, from pair `first` on, as they are or as f16
  const auto put = [&](int first, auto f16, auto pairs) {
    constexpr int kEach = f16.value ? 4 : 2;  // pairs in 16 bytes
#pragma unroll
    for (int i = 0; i < pairs.value / kEach; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (f16.value) {
          const Pair& q = v[first + 4 * i + j];
          const __half2 h = __floats2half2_rn(q.f[0], q.f[1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          w[j] = __float_as_uint(v[first + 2 * i + j / 2].f[j % 2]);
        }
      }
      mine[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __syncwarp();
  };
  using All = std::integral_constant<int, 16>;
  using Half = std::integral_constant<int, 8>;
  if (aligned) {
    put(0, std::bool_constant<kF16>{}, All{});
    constexpr int kPieces = kF16 ? 4 : 8, kRowsAtOnce = 32 / kPieces;  // of 16 bytes in a row
    const int r0 = lane / kPieces, piece = lane % kPieces;
    T* d = static_cast<T*>(p.y) + int64_t(m_base + r0) * p.ld_y + n;
#pragma unroll
    for (int i = 0; i < kPieces; ++i, d += kRowsAtOnce * p.ld_y) {
      const uint4 w = reinterpret_cast<const uint4*>(turn + (r0 + i * kRowsAtOnce) * kPitch<T>)[piece];
      if (m_base + r0 + i * kRowsAtOnce < p.m) reinterpret_cast<uint4*>(d)[piece] = w;
    }
    __syncwarp();
    return;
  }
  // Rows that start anywhere, or end inside the block: neighbours in neighbouring lanes, value by value,
  // eight rows in flight.  From what was put: rows of `each` lanes, U values `pitch` apart.
  const int rows = min(32, p.m - m_base);
  const auto take = [&](auto unit, int col0, auto lanes) {
    using U = decltype(unit);
    constexpr int kAtOnce = 32 / lanes.value, kRowPitch = kPitch<T> * 4 / sizeof(U) * kAtOnce;
    const int r0 = lane / lanes.value, c = n + col0 + lane % lanes.value;
    if (c < p.n) {
      T* d = static_cast<T*>(p.y) + int64_t(m_base + r0) * p.ld_y + c;
      const T* r = p.res ? static_cast<const T*>(p.res) + int64_t(m_base + r0) * p.ld_res + c : nullptr;
      const U* t = reinterpret_cast<const U*>(turn + r0 * kPitch<T>) + lane % lanes.value;
      for (int i = r0; i < rows; i += 8 * kAtOnce, t += 8 * kRowPitch) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = to_f32(t[j * kRowPitch]);
        if (r) {
          float add[8];
#pragma unroll
          for (int j = 0; j < 8; ++j, r += kAtOnce * p.ld_res)
            add[j] = i + j * kAtOnce < rows ? to_f32(*r) : 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = __fadd_rn(y[j], add[j]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j, d += kAtOnce * p.ld_y)
          if (i + j * kAtOnce < rows) *d = from_f32<T>(y[j]);
      }
    }
    __syncwarp();
  };
  if constexpr (!kF16) {
    put(0, std::false_type{}, All{});
    take(0.f, 0, std::integral_constant<int, 32>{});
  } else if (!p.res) {
    put(0, std::true_type{}, All{});
    take(T{}, 0, std::integral_constant<int, 32>{});
  } else {  // the sums are rounded once, with what is added: half of the columns at a time
    put(0, std::false_type{}, Half{});
    take(0.f, 0, std::integral_constant<int, 16>{});
    put(8, std::false_type{}, Half{});
    take(0.f, 16, std::integral_constant<int, 16>{});
  }
}

// What an epilogue warp multiplies an item's sums with: its token's scale, and by lane the scales of its
// blocks of columns and their biases or up scales.  Fetched an item ahead.
struct Ahead {
  float xs, ws[4], second[4];
};
template <bool GATE>
__device__ __forceinline__ Ahead look_ahead(const Q8Params& p, const Item& it, int m0, int warp,
                                            int lane) {
  Ahead a;
  const int m = m0 + (warp & 3) * 32 + lane, half = warp >> 2;
  const int blocks = (GATE ? it.bn / 2 : it.bn) / 32;
  a.xs = m < p.m ? p.xs[m] : 0.f;
#pragma unroll
  for (int i = 0; i < (GATE ? 2 : 4); ++i) {
    const int b = half + 2 * i, c = it.n0 + b * 32 + lane;
    const bool there = b < blocks && c < p.n;
    a.ws[i] = there ? p.ws[c] : 0.f;
    if constexpr (GATE) a.second[i] = there ? p.us[c] : 0.f;
    else a.second[i] = there && p.bias ? p.bias[c] : 0.f;
  }
  return a;
}

// A row's 32 values of what is added to a block, where it can be read in whole pieces.
template <class T>
struct Addend {
  static constexpr int V = 16 / sizeof(T), kPieces = 32 / V;
  union {
    uint4 u;
    T e[V];
  } w[kPieces];
};
template <class T>
__device__ __forceinline__ void load_addend(Addend<T>& a, const Q8Params& p, int m, int n) {
  if (p.res && p.wide && n + 32 <= p.n && m < p.m) {
    const uint4* r = reinterpret_cast<const uint4*>(static_cast<const T*>(p.res) +
                                                    int64_t(m) * p.ld_res + n);
#pragma unroll
    for (int j = 0; j < Addend<T>::kPieces; ++j) a.w[j].u = r[j];
  } else {
#pragma unroll
    for (int j = 0; j < Addend<T>::kPieces; ++j) a.w[j].u = make_uint4(0, 0, 0, 0);
  }
}

// The epilogue of one item by epilogue warp `warp`: TMEM lane quarter warp & 3, every other block of 32
// columns.
template <class T, bool GATE, class Release>
__device__ __forceinline__ void wide_epilogue(const Q8Params& p, WideSmem<T>& s, uint32_t acc,
                                              const Item& it, int m0, const Ahead& ahead,
                                              Addend<T>& addend, int warp, int lane,
                                              Release release) {
  const int quarter = warp & 3, half = warp >> 2;
  const int cols = GATE ? it.bn / 2 : it.bn, blocks = cols / 32;
  const uint32_t at = acc + (uint32_t(quarter * 32) << 16);
  const int m_base = m0 + quarter * 32;
  const float* ws = s.col[warp][0];
  const float* second = s.col[warp][1];
  const Pair xs2 = pair(ahead.xs, ahead.xs);
  const int m = m_base + lane;
  for (int b = half, i = 0; b < blocks; b += 2, i += 32) {
    const int n = it.n0 + b * 32;
    const bool some = m_base < p.m && n < p.n, aligned = p.wide && n + 32 <= p.n;
    const bool add = !GATE && p.res && aligned;
    Addend<T> now;
    if constexpr (!GATE) {
      now = addend;
      if (p.res && b + 2 < blocks) load_addend(addend, p, m, n + 64);
    }
    uint32_t r[32], ru[GATE ? 32 : 1];
    Pair v[16];
    tmem_ld32(at + b * 32, r);
    if constexpr (GATE) tmem_ld32(at + cols + b * 32, ru);
    tmem_ld_wait();
    if (b + 2 >= blocks) {  // everything of this warp is in registers
      tc_fence_before();
      __syncwarp();
      release();
    }
    const float4* w4 = reinterpret_cast<const float4*>(ws + i);
    const float4* s4 = reinterpret_cast<const float4*>(second + i);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 w = w4[j];
      v[2 * j] = scaled2(r[4 * j], r[4 * j + 1], xs2, pair(w.x, w.y));
      v[2 * j + 1] = scaled2(r[4 * j + 2], r[4 * j + 3], xs2, pair(w.z, w.w));
    }
    if constexpr (GATE) {
      const auto finish = [&](auto gelu) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 w = s4[j];
          v[2 * j] = act_mul<gelu.value>(
              v[2 * j], scaled2(ru[4 * j], ru[4 * j + 1], xs2, pair(w.x, w.y)));
          v[2 * j + 1] = act_mul<gelu.value>(
              v[2 * j + 1], scaled2(ru[4 * j + 2], ru[4 * j + 3], xs2, pair(w.z, w.w)));
        }
      };
      if (p.act == kActSilu) finish(std::false_type{});
      else finish(std::true_type{});
    } else if (p.bias) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 w = s4[j];
        v[2 * j] = add2(v[2 * j], pair(w.x, w.y));
        v[2 * j + 1] = add2(v[2 * j + 1], pair(w.z, w.w));
      }
    }
    if constexpr (!GATE) {
      constexpr int V = Addend<T>::V;
      if (add) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          v[j] = add2(v[j], pair(to_f32(now.w[2 * j / V].e[2 * j % V]),
                                 to_f32(now.w[2 * j / V].e[2 * j % V + 1])));
      }
    }
    if (some) store_block<T>(p, v, m_base, lane, n, aligned, s.turn[warp]);
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
  constexpr uint32_t kStages = kWideStages<T>;
  WideSmem<T>& s = *reinterpret_cast<WideSmem<T>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                   ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = int(cluster_id_x()), pairs = int(cluster_count_x());
  const int nk = (p.k + kStep - 1) / kStep;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
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
    // the whole warp walks the ring, so that what the copies take is the same in all its lanes
    const CUtensorMap* tm_b = GATE && rank ? &tm_u : &tm_w;
    uint32_t st = 0, round = 0;
    bool ok = true;
    for (int i = pair; i < p.items && ok; i += pairs) {
      const Item it = item_of<GATE>(p, i);
      const int m0 = it.m0 + int(rank) * kRows, half = it.bn / 2;
      const int n0 = GATE ? it.n0 : it.n0 + int(rank) * half;
      for (int kt = 0; kt < nk; ++kt) {
        if (round > 0 && !(ok = gemm_wait_all(s.abort_flag, &s.empty[st], (round - 1) & 1, p.err)))
          break;
        if (elect_one()) {
          const uint32_t full0 = cluster_map(smem_u32(&s.full[st]), 0);
          if (rank == 0)
            mbar_arrive_expect_tx(&s.full[st], 2 * (kTileBytes + half * kStep) +
                                                   (st + round == 0 ? p.wait_deficit : 0));
          tma_load_3d_pair(s.a[st], &tm_x, kt * kStep, m0, 0, full0);
          tma_load_3d_pair(s.b[st], tm_b, kt * kStep, n0, 0, full0);
          if (half > kBoxRows)
            tma_load_3d_pair(s.b[st] + kBoxRows * kStep, tm_b, kt * kStep, n0 + kBoxRows, 0, full0);
        }
        __syncwarp();
        if (++st == kStages) {
          st = 0;
          ++round;
        }
      }
    }
    if (!ok && lane == 0) {  // let the copies already in flight land before the CTA exits
      if (rank == 0) {
        for (int h = 0; h < kStages; ++h) {
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(&s.full[h], uint32_t(h) < st ? round & 1 : (round - 1) & 1) &&
                 globaltimer_ns() - t0 < kGemmWaitNs) {
          }
        }
      } else {  // its loads complete on the even CTA's barriers: give them time to land
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 100000) {
        }
      }
    }
    __syncwarp();
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
            !(ok = gemm_wait_all(s.abort_flag, &s.acc_empty[b], (u - 1) & 1, p.err)))
          break;
        tc_fence_after();
        const uint32_t idesc = idesc_i8(2 * kRows, item_of<GATE>(p, i).bn);
        const uint32_t acc = tmem + uint32_t(b * kWidth);
        for (int kt = 0; kt < nk; ++kt, ++g) {
          const uint32_t st = g % kStages;
          if (!(ok = gemm_wait_all(s.abort_flag, &s.full[st], (g / kStages) & 1, p.err)))
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
    Ahead ahead{};
    if (pair < p.items) {
      const Item it = item_of<GATE>(p, pair);
      ahead = look_ahead<GATE>(p, it, it.m0 + int(rank) * kRows, warp, lane);
    }
    for (int i = pair; i < p.items; i += pairs, ++n) {
      const int b = n & 1, u = n >> 1;
      const Item it = item_of<GATE>(p, i);
      const Ahead now = ahead;
      __syncwarp();
#pragma unroll
      for (int j = 0; j < (GATE ? 2 : 4); ++j) {
        s.col[warp][0][32 * j + lane] = now.ws[j];
        s.col[warp][1][32 * j + lane] = now.second[j];
      }
      __syncwarp();
      if (i + pairs < p.items) {
        const Item next = item_of<GATE>(p, i + pairs);
        ahead = look_ahead<GATE>(p, next, next.m0 + int(rank) * kRows, warp, lane);
      }
      Addend<T> addend;  // of the first block, on its way while the MMAs run
      if constexpr (!GATE)
        if (p.res)
          load_addend(addend, p, it.m0 + int(rank) * kRows + (warp & 3) * 32 + lane,
                      it.n0 + (warp >> 2) * 32);
      if (!gemm_wait_all(s.abort_flag, &s.acc_full[b], u & 1, p.err)) break;
      tc_fence_after();
      const uint32_t empty0 = cluster_map(smem_u32(&s.acc_empty[b]), 0);
      // TMEM loads are ordered by the fence in front of the arrival; nothing else is guarded by it
      wide_epilogue<T, GATE>(p, s, tmem + uint32_t(b * kWidth), it, it.m0 + int(rank) * kRows, now,
                             addend, warp, lane, [&] {
                               if (lane == 0) mbar_arrive_cluster_relaxed(empty0);
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
// The weights' bytes bound these calls, so the weights are the MMA's rows: a tile is `rows` channels (any
// multiple of 8 up to 128, so that the tiles fill the SMs evenly; the MMA's rows behind them hold whatever
// lies there and are not looked at) times up to kMostTokens tokens.  GATE: two products of the same
// tokens, whose sums lie in the same TMEM lanes.  A persistent CTA per SM walks tiles, its ring and two
// accumulators running on across them.
//   SPLIT: too few channels for that; a tile's k is cut over a cluster, one tile each.  Every CTA sums its
// part and hands the sums, by token, to the CTA that finishes that token.
constexpr int kNarrowEpi = 8;        // epilogue warps: two per TMEM lane quarter
constexpr int kNarrowThreads = 32 * (2 + kNarrowEpi);  // TMA, MMA, epilogue
constexpr int kMostTokens = 128;     // of a tile
constexpr int kMostNarrow = 2048;    // of a call
constexpr int kMostSplit = 8;
constexpr int kMostStages = 24;
constexpr int kNarrowSmem = 226 * 1024;

struct NarrowHead {  // in front of the ring and the sums
  uint64_t full[kMostStages], empty[kMostStages];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t done;
  uint32_t tmem_base;
  volatile int abort_flag;
};
static_assert(sizeof(NarrowHead) <= 1024, "the head is one swizzle atom");

__device__ __forceinline__ void st_cluster4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                            uint32_t d) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

__host__ __device__ inline int split_tokens(int tokens, int split) {
  return ((tokens + split - 1) / split + 3) / 4 * 4;
}
// TMEM is allocated in powers of two.
__host__ __device__ inline uint32_t tmem_columns(uint32_t need) {
  return need <= 32 ? 32 : need <= 64 ? 64 : need <= 128 ? 128 : need <= 256 ? 256 : 512;
}

template <class T, bool GATE, bool SPLIT>
__global__ void __launch_bounds__(kNarrowThreads, 1)
    narrow_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                  const __grid_constant__ CUtensorMap tm_u, const __grid_constant__ Q8Params p) {
  constexpr int G = GATE ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  NarrowHead& s = *reinterpret_cast<NarrowHead*>(base);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = SPLIT ? int(cluster_ctas()) : 1, rank = SPLIT ? int(cluster_ctarank()) : 0;
  const int first = SPLIT ? int(blockIdx.x) / split : int(blockIdx.x);
  const int step = SPLIT ? p.items : int(gridDim.x);
  // a stage: `chunks` steps of k, [w][chunk][rows][128], GATE: [up] likewise, [x][chunk][tokens][128]
  const uint32_t w_step = uint32_t(p.rows) * kStep, x_step = uint32_t(p.tokens) * kStep;
  const uint32_t w_bytes = p.chunks * w_step, stage_bytes = G * w_bytes + p.chunks * x_step;
  // SPLIT: tokens finished here, in fours, and where the sums lie: [split][G][rows][own + 4] (the four words
  // between two channels keep 16-byte accesses of neighbouring channels free of conflicts)
  const int own = split_tokens(p.tokens, split), pitch = own + 4;
  uint32_t* sums = reinterpret_cast<uint32_t*>(base + 1024);
  constexpr int kScales = kNarrowEpi * kMostTokens * 4;  // each epilogue warp's copy of the tokens' scales
  uint8_t* ring = base + 1024 + (SPLIT ? (split * G * p.rows * pitch * 4 + 1023) / 1024 * 1024 : kScales);
  const int nk = p.steps;  // stages of a tile
  const int k0 = SPLIT ? nk * rank / split : 0, k1 = SPLIT ? nk * (rank + 1) / split : nk;
  const uint32_t acc_cols = G * p.tokens;  // of one accumulator buffer
  const uint32_t need = SPLIT ? acc_cols : 2 * acc_cols;
  const uint32_t tmem_cols = tmem_columns(need);
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.acc_full[i], 1);
      mbar_init(&s.acc_empty[i], kNarrowEpi);
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
  if constexpr (SPLIT) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  grid_dependency_wait();
  launch_dependents();

  // SPLIT: what the epilogue warps finish: blocks of 32 channels, a block a warp (or several, each every
  // so many tokens); scales and biases are fetched now.
  const int n0 = first % p.tiles_n * p.rows, m0 = first / p.tiles_n * p.tokens;
  const int blocks = (p.rows + 31) / 32, groups = kNarrowEpi / blocks, group = (warp - 2) / blocks;
  const int mine = min(own, min(p.tokens, p.m - m0) - rank * own);  // tokens to finish
  int ln = -1;  // this lane's channel of the tile, if it has one
  float ws = 0.f, second = 0.f;
  if (SPLIT && warp >= 2 && group < groups) {
    ln = (warp - 2) % blocks * 32 + lane;
    if (ln >= p.rows || n0 + ln >= p.n) ln = -1;
    if (ln >= 0) {
      ws = p.ws[n0 + ln];
      if constexpr (GATE) second = p.us[n0 + ln];
      else if (p.bias) second = p.bias[n0 + ln];
    }
    if (lane < mine) asm volatile("prefetch.global.L1 [%0];" ::"l"(p.xs + m0 + rank * own + lane));
  }

  if (warp == 0) {
    // the whole warp walks the ring, so that what the copies take is the same in all its lanes
    uint32_t st = 0, round = 0;
    bool ok = true;
    for (int t = first; t < p.items && ok; t += step) {
      const int n0 = t % p.tiles_n * p.rows, m0 = t / p.tiles_n * p.tokens;
      // each CTA begins at another part of k, since all of them read the same tokens (gate and up of one
      // token, 2 x 8192 x 2048: 0.3 of 7 us less than with all of them at the same part)
      int kt = k0 + first % (k1 - k0);
      for (int i = k0; i < k1; ++i) {
        if (round > 0 && !(ok = gemm_wait_all(s.abort_flag, &s.empty[st], (round - 1) & 1, p.err)))
          break;
        if (elect_one()) {
          uint8_t* a = ring + st * stage_bytes;
          const int kx = p.deep ? 0 : kt * kStep, kz = p.deep ? kt * p.chunks : 0;
          mbar_arrive_expect_tx(&s.full[st], stage_bytes + (st + round == 0 ? p.wait_deficit : 0));
          tma_load_3d(a, &tm_w, kx, n0, kz, &s.full[st]);
          if constexpr (GATE) tma_load_3d(a + w_bytes, &tm_u, kx, n0, kz, &s.full[st]);
          tma_load_3d(a + G * w_bytes, &tm_x, kx, m0, kz, &s.full[st]);
        }
        __syncwarp();
        if (++kt == k1) kt = k0;
        if (++st == uint32_t(p.stages)) {
          st = 0;
          ++round;
        }
      }
    }
    if (!ok && lane == 0) {  // let the copies already in flight land before the CTA exits: those of this
                             // round in front of st, those of the one before from st on
      for (int h = 0; h < p.stages; ++h) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&s.full[h], uint32_t(h) < st ? round & 1 : (round - 1) & 1) &&
               globaltimer_ns() - t0 < kGemmWaitNs) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t idesc = idesc_i8(p.rows <= 64 ? 64 : 128, p.tokens);
    const uint64_t desc0 = smem_desc_sw128(smem_u32(ring), 16, 1024);
    bool ok = true, issued = false;
    uint32_t st = 0, round = 0;
    int n = 0;  // tiles of this CTA
    for (int t = first; t < p.items && ok; t += step, ++n) {
      const int b = n & 1, u = n >> 1;  // accumulator buffer, its use count
      if (u > 0 && !(ok = gemm_wait_all(s.abort_flag, &s.acc_empty[b], (u - 1) & 1, p.err)))
        break;
      tc_fence_after();
      const uint32_t acc = tmem + uint32_t(b) * acc_cols;
      for (int kt = k0; kt < k1; ++kt) {
        if (!(ok = gemm_wait_all(s.abort_flag, &s.full[st], round & 1, p.err))) break;
        tc_fence_after();
        if (elect_one()) {
          uint64_t ad = desc0 + uint64_t(st) * (stage_bytes >> 4), bd = ad + ((G * w_bytes) >> 4);
          uint32_t more = kt > k0 ? 1u : 0u;
          for (int c = 0; c < p.chunks; ++c, ad += w_step >> 4, bd += x_step >> 4) {
#pragma unroll
            for (int kk = 0; kk < kStep / 32; ++kk) {
              mma_i8_ss(acc, ad + 2 * kk, bd + 2 * kk, idesc, more);
              if constexpr (GATE)
                mma_i8_ss(acc + p.tokens, ad + (w_bytes >> 4) + 2 * kk, bd + 2 * kk, idesc, more);
              more = 1u;
            }
          }
          mma_commit(&s.empty[st]);
        }
        issued = true;
        __syncwarp();
        if (++st == uint32_t(p.stages)) {
          st = 0;
          ++round;
        }
      }
      if (ok && elect_one()) mma_commit(&s.acc_full[b]);
      __syncwarp();
    }
    if (issued) {  // no MMA may still run when the TMEM is freed
      if (elect_one()) mma_commit(&s.done);
      __syncwarp();
      if (lane == 0) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&s.done, 0) && globaltimer_ns() - t0 < kGemmWaitNs) {
        }
      }
      __syncwarp();
    }
  } else {
    // lane of TMEM quarter warp & 3 -> channel: 32 a quarter, or 16 of an MMA of 64 rows.  The two warps of
    // a quarter take every other eight tokens.
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const bool tall = p.rows > 64;
    const int ch = tall ? quarter * 32 + lane : quarter * 16 + lane;
    const bool held = ch < p.rows && (tall || lane < 16);
    float* scales = reinterpret_cast<float*>(base + 1024) + (warp - 2) * kMostTokens;
    int n = 0, have = -1;  // tiles of this CTA; first token of the tile whose scales are there
    for (int t = first; t < p.items; t += step, ++n) {
      const int b = n & 1, u = n >> 1;
      const int c = t % p.tiles_n * p.rows + ch, m0 = t / p.tiles_n * p.tokens;
      const int tokens = min(p.tokens, p.m - m0);
      const bool live = held && c < p.n;
      float ws = 0.f, second = 0.f;
      if constexpr (!SPLIT) {
        if (live) {
          ws = p.ws[c];
          if constexpr (GATE) second = p.us[c];
          else if (p.bias) second = p.bias[c];
        }
        if (have != m0) {
          __syncwarp();
          for (int i = lane; i < p.tokens; i += 32) scales[i] = i < tokens ? p.xs[m0 + i] : 0.f;
          have = m0;
        }
      }
      __syncwarp();
      const bool ok = gemm_wait_all(s.abort_flag, &s.acc_full[b], u & 1, p.err);
      if constexpr (SPLIT) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      if (!ok) break;
      tc_fence_after();
      const uint32_t at = tmem + uint32_t(b) * acc_cols + (uint32_t(quarter * 32) << 16);
      if constexpr (SPLIT) {
        for (int t0 = half * 8; t0 < p.tokens; t0 += 16) {
          uint32_t r[G][8];
#pragma unroll
          for (int g = 0; g < G; ++g) tmem_ld8(at + g * p.tokens + t0, r[g]);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; j += 4) {
            const int to = (t0 + j) / own, tl = t0 + j - to * own;  // number tl of CTA `to`
            const uint32_t dst = cluster_map(
                smem_u32(sums + (rank * G * p.rows + ch) * pitch + tl), uint32_t(to));
#pragma unroll
            for (int g = 0; g < G; ++g)
              if (held)
                st_cluster4(dst + g * p.rows * pitch * 4, r[g][j], r[g][j + 1], r[g][j + 2], r[g][j + 3]);
          }
        }
      } else {
        const Pair ws2 = pair(ws, ws), second2 = pair(second, second);
        T* y = static_cast<T*>(p.y) + int64_t(m0 + half * 8) * p.ld_y + c;
        const T* res = p.res ? static_cast<const T*>(p.res) + int64_t(m0 + half * 8) * p.ld_res + c : nullptr;
        for (int t0 = half * 8; t0 < p.tokens; t0 += 16) {
          const int left = tokens - t0;  // of these eight
          uint32_t r[G][8];
#pragma unroll
          for (int g = 0; g < G; ++g) tmem_ld8(at + g * p.tokens + t0, r[g]);
          float add[8];
          if (!GATE && res) {
            const T* q = res;
#pragma unroll
            for (int j = 0; j < 8; ++j, q += p.ld_res) add[j] = live && j < left ? to_f32(*q) : 0.f;
            res += 16 * p.ld_res;
          }
          tmem_ld_wait();
          if (t0 + 16 >= p.tokens) {  // everything of this warp is in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.acc_empty[b]);
          }
          T* d = y;
#pragma unroll
          for (int j = 0; j < 8; j += 2, d += 2 * p.ld_y) {
            const Pair xs2 = pair(scales[t0 + j], scales[t0 + j + 1]);
            Pair v = scaled2(r[0][j], r[0][j + 1], xs2, ws2);
            if constexpr (GATE) {
              v = act_mul(v, scaled2(r[G - 1][j], r[G - 1][j + 1], xs2, second2), p.act);
            } else {
              if (p.bias) v = add2(v, second2);
              if (res) v = add2(v, pair(add[j], add[j + 1]));
            }
            if (live && j < left) d[0] = from_f32<T>(v.f[0]);
            if (live && j + 1 < left) d[p.ld_y] = from_f32<T>(v.f[1]);
          }
          y += 16 * p.ld_y;
        }
        // a tile of eight tokens has none for the second warp of a quarter
        if (half * 8 >= p.tokens && lane == 0) mbar_arrive(&s.acc_empty[b]);
      }
    }
  }

  if constexpr (SPLIT) {
    if (warp < 2) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (s.abort_flag && lane == 0)  // nothing of a sum that lacks a part is stored
      for (int i = 0; i < split; ++i)
        st_cluster(cluster_map(smem_u32(const_cast<int*>(&s.abort_flag)), i), 1u);
    tc_fence_before();
    cluster_sync();
  } else {
    tc_fence_before();
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
  if constexpr (SPLIT) {
    if (s.abort_flag || warp < 2) return;
    if (ln >= 0) {
      const int n = n0 + ln;
      T* y = static_cast<T*>(p.y) + int64_t(m0 + rank * own) * p.ld_y + n;
      const T* res = static_cast<const T*>(p.res) + int64_t(m0 + rank * own) * p.ld_res + n;
      const Pair ws2 = pair(ws, ws), second2 = pair(second, second);
      for (int tl = 4 * group; tl < mine; tl += 4 * groups) {
        Pair xs[2];
        float add[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          xs[j / 2].f[j % 2] = tl + j < mine ? p.xs[m0 + rank * own + tl + j] : 0.f;
          add[j] = !GATE && p.res && tl + j < mine ? to_f32(res[int64_t(tl + j) * p.ld_res]) : 0.f;
        }
        int acc[G][4] = {};
        const uint32_t* q = sums + ln * pitch + tl;
        for (int k = 0; k < split; ++k)
#pragma unroll
          for (int g = 0; g < G; ++g, q += p.rows * pitch) {
            const uint4 a = *reinterpret_cast<const uint4*>(q);
            acc[g][0] += int(a.x);
            acc[g][1] += int(a.y);
            acc[g][2] += int(a.z);
            acc[g][3] += int(a.w);
          }
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          Pair v = scaled2(acc[0][j], acc[0][j + 1], xs[j / 2], ws2);
          if constexpr (GATE) {
            v = act_mul(v, scaled2(acc[G - 1][j], acc[G - 1][j + 1], xs[j / 2], second2), p.act);
          } else {
            if (p.bias) v = add2(v, second2);
            if (p.res) v = add2(v, pair(add[j], add[j + 1]));
          }
          if (tl + j < mine) y[int64_t(tl + j) * p.ld_y] = from_f32<T>(v.f[0]);
          if (tl + j + 1 < mine) y[int64_t(tl + j + 1) * p.ld_y] = from_f32<T>(v.f[1]);
        }
      }
    }
  }
}

// ---- host -------------------------------------------------------------------------------------------
// Rows of codes in boxes of 128 codes x box_rows, 128-byte swizzle; what lies outside reads as 0.
// chunks > 1: rows of whole steps of 128 codes, the steps a dimension of their own, that many of them in
// a box.
bool map_codes(CUtensorMap* m, const Q8Rows& r, int box_rows, int chunks = 1) {
  auto enc = encode_fn();
  if (!enc) return false;
  const bool deep = chunks > 1;
  cuuint64_t dims[3] = {cuuint64_t(deep ? kStep : r.cols), cuuint64_t(r.rows),
                        cuuint64_t(deep ? r.cols / kStep : 1)};
  cuuint64_t strides[2] = {cuuint64_t(r.ld), kStep};
  cuuint32_t box[3] = {kStep, cuuint32_t(box_rows), cuuint32_t(chunks)};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, r.q, dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
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

// Tiles of wide_kernel: the last wave's are halved where their halves still fit one wave.
struct WideItems {
  int64_t tiles_n, tiles, whole, items;
};
WideItems wide_items(int m, int n, int G, int pairs) {
  const int cols = kWidth / G;
  WideItems w;
  w.tiles_n = (int64_t(n) + cols - 1) / cols;
  w.tiles = w.tiles_n * ((int64_t(m) + 2 * kRows - 1) / (2 * kRows));
  const int64_t rest = w.tiles % pairs;
  w.whole = 2 * rest <= pairs ? w.tiles - rest : w.tiles;
  w.items = w.whole + 2 * (w.tiles - w.whole);
  return w;
}

template <class T, bool GATE>
cudaError_t launch_wide(Q8Params p, const GemmQ8Args& a, int num_sms, cudaStream_t stream) {
  CUtensorMap tx, tw, tu;
  if (!map_codes(&tx, a.x, kRows) || !map_codes(&tw, a.w, kBoxRows) ||
      !map_codes(&tu, GATE ? a.up : a.w, kBoxRows))
    return cudaErrorInvalidValue;
  const void* fn = reinterpret_cast<const void*>(&wide_kernel<T, GATE>);
  const size_t smem = sizeof(WideSmem<T>) + 1024;
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
  const WideItems w = wide_items(p.m, p.n, GATE ? 2 : 1, max_pairs);
  if (2 * w.tiles > INT32_MAX) return cudaErrorInvalidValue;
  p.tiles_n = int32_t(w.tiles_n);
  p.whole = int32_t(w.whole);
  p.items = int32_t(w.items);
  void* args[] = {&tx, &tw, &tu, &p};
  return launch_cluster(fn, 2 * std::min<int64_t>(p.items, max_pairs), kWideThreads, smem, 2, args,
                        stream);
}

// How few tokens are cut up.
struct NarrowPlan {
  int rows, tokens, split;  // channels and tokens of a tile, CTAs of its k
  int chunks, steps;        // steps of 128 codes in a stage, stages of a tile
  float cost;               // cycles
};
// Clusters of 2, 4 and 8 CTAs, one CTA an SM, that run at once (148 SMs in groups that hold no multiple of
// 8): 8 bits each.
cudaError_t cluster_room(int* room) {
  static PerDeviceOnce setup;
  return per_device_once(setup, [](int& packed) {
    const void* fn = reinterpret_cast<const void*>(&narrow_kernel<__half, false, true>);
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kNarrowSmem);
    for (int i = 0; i < 3 && e == cudaSuccess; ++i) {
      cudaLaunchAttribute at{};
      at.id = cudaLaunchAttributeClusterDimension;
      at.val.clusterDim.x = 2u << i;
      at.val.clusterDim.y = 1;
      at.val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(2u << i);
      cfg.blockDim = dim3(kNarrowThreads);
      cfg.dynamicSmemBytes = kNarrowSmem;
      cfg.attrs = &at;
      cfg.numAttrs = 1;
      int n = 0;
      e = cudaOccupancyMaxActiveClusters(&n, fn, &cfg);
      packed |= std::min(std::max(n, 1), 255) << (8 * i);
    }
    return e;
  }, room);
}
// The busiest SM's time, from what was measured over rows 16 to 128 of 8 to 128 tokens: a stage takes the
// longest of its bytes at 50 a cycle, its weights' at an SM's share of the DRAM rate (23 where all SMs
// load), and its MMAs (8192 products a cycle with 128 rows, half with 64), and 150 more; or the MMAs'
// issue, 37 cycles each and 260 to hand the stage over.  The last tile's epilogue, or the exchange of a
// cluster's sums, follows.
NarrowPlan narrow_plan(int m, int n, int k, int G, int num_sms, int room) {
  constexpr float kLoad = 50, kDram = 23, kWait = 150, kIssue = 37, kHandOver = 260;
  constexpr int kMostChunks = 4, kMostStage = 64 * 1024;
  // the MMA's columns: 8 or a multiple of 16, with 64 rows also 24 (which not every list of kind::i8's shapes
  // has; 20 x 2048 x 2048 4.6 us, 4.8 with 32)
  const int fewest = std::min(kMostTokens, m <= 24 ? (m + 7) / 8 * 8 : (m + 15) / 16 * 16);
  const int token_tiles = (m + fewest - 1) / fewest, nk = (k + kStep - 1) / kStep;
  const float sms = float(num_sms);
  NarrowPlan best{};
  for (int rows = 8; rows <= 128; rows += 8) {
    const int tokens = rows > 64 && fewest > 8 ? (fewest + 15) / 16 * 16 : fewest;
    const float mma = 4.f * G * tokens / 2.f;
    const int64_t tiles = (int64_t(n) + rows - 1) / rows * token_tiles;
    const float all = (G * rows + tokens) * kStep / kLoad, weights = float(G * rows * kStep);
    for (int split = 1, i = 0; split <= std::min(kMostSplit, nk); split *= 2, ++i) {
      if (split > 1 && G * rows > 128) break;
      const int slots = split > 1 ? (room >> (8 * (i - 1))) & 255 : num_sms;
      const float busy = float(std::min<int64_t>(tiles, slots) * split) / sms;
      const float bytes = std::max({all, weights / std::min(kLoad, kDram / busy), mma});
      const float turns = float((tiles + slots - 1) / slots);
      const float fixed = split > 1 ? turns * (1300 + 0.52f * G * rows * tokens + 12 * tokens)
                                    : turns * 100 + 30.f * tokens;
      for (int chunks = kMostChunks; chunks >= 1; --chunks) {
        // stages of several steps want rows of whole steps, and leave no part of a stage empty
        if (chunks > 1 &&
            (k % kStep || nk % chunks || chunks * (G * rows + tokens) * kStep > kMostStage))
          continue;
        const int steps = nk / chunks;
        if (split > steps) continue;
        const float stage = std::max(chunks * bytes + kWait, chunks * 4 * G * kIssue + kHandOver);
        const float cost = turns * ((steps + split - 1) / split) * stage + fixed;
        if (!best.rows || cost < best.cost) best = NarrowPlan{rows, tokens, split, chunks, steps, cost};
        if (steps % split == 0) break;  // smaller stages only wait more often
      }
    }
  }
  return best;
}
// The same of wide_kernel: a step of a whole tile takes 512 cycles, of half a tile 305; pairs of CTAs start
// later.
double wide_cost(int m, int n, int k, int G, int num_sms) {
  const int cols = kWidth / G, pairs = std::max(1, num_sms / 2), nk = (k + kStep - 1) / kStep;
  const int64_t tiles = (int64_t(n) + cols - 1) / cols * ((m + 2 * kRows - 1) / (2 * kRows));
  const int64_t rest = tiles % pairs;
  const double whole = double(tiles / pairs + (2 * rest > pairs ? 1 : 0));
  return 4000 + nk * (512 * whole + (rest && 2 * rest <= pairs ? 305 : 0));
}

// What a CTA of that plan takes of its SM.
struct NarrowRoom {
  int stages;  // of the ring
  int smem;    // bytes of shared memory asked for
  int cols;    // of TMEM
};
constexpr int kSmemOfSm = 228 * 1024, kKeptOfCta = 1024, kTmemOfSm = 512;  // (kept for the system)
constexpr int kSplitSmem = 48 * 1024;  // a split CTA's at least
// The CTAs of a cluster wait for one another, without a bound, and an allocation of TMEM waits for whoever
// holds the columns.  So the CTAs of clusters that fit on one SM by their shared memory, of any calls on any
// streams, must find their columns there: a split CTA asks for at least its columns' share of the SM's
// shared memory (56 KB and the 1 KB kept of each CTA for 128 columns, 113 for 256), and for more than a pair
// form's CTA, which takes all columns, leaves of it.  (An unsplit CTA waits for nobody that waits for it.)
NarrowRoom narrow_room(const NarrowPlan& plan, int G, int64_t tiles, int num_sms) {
  const bool split = plan.split > 1;
  const int own = split_tokens(plan.tokens, plan.split);
  const int stage = (G * plan.rows + plan.tokens) * kStep * plan.chunks;
  const int sums = split ? (plan.split * G * plan.rows * (own + 4) * 4 + 1023) / 1024 * 1024
                         : kNarrowEpi * kMostTokens * 4;
  // behind the ring, what the last stage's MMA reads beyond its rows
  const int fixed = 2048 + sums + (plan.rows <= 64 ? 64 : 128) * kStep;
  const int64_t steps = split ? (plan.steps + plan.split - 1) / plan.split
                              : plan.steps * ((tiles + num_sms - 1) / num_sms);
  NarrowRoom r;
  r.stages = int(std::min<int64_t>({kMostStages, steps, (kNarrowSmem - fixed) / stage}));
  r.cols = int(tmem_columns((split ? 1 : 2) * G * plan.tokens));
  r.smem = fixed + r.stages * stage;
  if (split) r.smem = std::max({r.smem, kSplitSmem, r.cols * (kSmemOfSm / kTmemOfSm) - kKeptOfCta});
  return r;
}
static_assert(sizeof(WideSmem<__half>) + kSplitSmem > kSmemOfSm &&
                  sizeof(WideSmem<float>) + kSplitSmem > kSmemOfSm,
              "no split CTA beside a pair form's");

template <class T, bool GATE, bool SPLIT>
cudaError_t launch_narrow(Q8Params p, const GemmQ8Args& a, const NarrowPlan& plan, int num_sms,
                          cudaStream_t stream) {
  constexpr int G = GATE ? 2 : 1;
  CUtensorMap tx, tw, tu;
  if (!map_codes(&tx, a.x, plan.tokens, plan.chunks) || !map_codes(&tw, a.w, plan.rows, plan.chunks) ||
      (GATE && !map_codes(&tu, a.up, plan.rows, plan.chunks)))
    return cudaErrorInvalidValue;
  if (!GATE) tu = tw;
  p.rows = plan.rows;
  p.tokens = plan.tokens;
  p.steps = plan.steps;
  p.chunks = plan.chunks;
  p.deep = plan.chunks > 1;
  p.tiles_n = (p.n + plan.rows - 1) / plan.rows;
  const int64_t tiles = int64_t(p.tiles_n) * ((int64_t(p.m) + plan.tokens - 1) / plan.tokens);
  if (tiles * plan.split > INT32_MAX) return cudaErrorInvalidValue;
  p.items = int32_t(tiles);
  const NarrowRoom need = narrow_room(plan, G, tiles, num_sms);
  p.stages = need.stages;
  const void* fn = reinterpret_cast<const void*>(&narrow_kernel<T, GATE, SPLIT>);
  static PerDeviceOnce attrs;
  cudaError_t e = per_device_once(attrs, [&](int&) {
    return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kNarrowSmem);
  });
  if (e != cudaSuccess) return e;
  void* args[] = {&tx, &tw, &tu, &p};
  return launch_cluster(fn, SPLIT ? tiles * plan.split : std::min<int64_t>(tiles, num_sms),
                        kNarrowThreads, size_t(need.smem), plan.split, args, stream);
}

bool on16(const void* p, int64_t pitch_bytes) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && pitch_bytes % 16 == 0;
}

// Which of the two kernels, and how.
struct Choice {
  bool wide;
  NarrowPlan plan;
};
Choice choose(int m, int n, int k, int G, int num_sms, int room) {
  Choice c{m > kMostNarrow, {}};
  if (c.wide) return c;
  c.plan = narrow_plan(m, n, k, G, num_sms, room);
  c.wide = m > kMostTokens && c.plan.cost > wide_cost(m, n, k, G, num_sms);
  return c;
}

template <class T, bool GATE>
cudaError_t launch_q8(const Q8Params& p, const GemmQ8Args& a, int num_sms, cudaStream_t s) {
  constexpr int G = GATE ? 2 : 1;
  int room = 0;
  if (p.m <= kMostNarrow) {
    const cudaError_t e = cluster_room(&room);
    if (e != cudaSuccess) return e;
  }
  const Choice c = choose(p.m, p.n, p.k, G, num_sms, room);
  if (c.wide) return launch_wide<T, GATE>(p, a, num_sms, s);
  return c.plan.split > 1 ? launch_narrow<T, GATE, true>(p, a, c.plan, num_sms, s)
                          : launch_narrow<T, GATE, false>(p, a, c.plan, num_sms, s);
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
  p.wait_deficit = a.wait_deficit;
  const int64_t es = dtype == 0 ? 2 : 4;
  p.wide = on16(a.y, a.ld_y * es) && (!a.res || on16(a.res, a.ld_res * es));
  if (a.up.q) return launch_q8<__half, true>(p, a, num_sms, s);
  return dtype == 0 ? launch_q8<__half, false>(p, a, num_sms, s)
                    : launch_q8<float, false>(p, a, num_sms, s);
}

}  // namespace p2p
