// rows_q8.cu -- rows of 8-bit integers with a scale each: made from f16 / f32 rows, alone or behind
// the residual addition and RMS norm of a decoder layer (ADD_RMS,
// src/scripts/lfm-engine/kernels.js:146-182), and read back as values (the embedding lookup).
//
// All three move bytes: a row is read once, kept in registers, reduced and written once.  A code is
// 127 v / a, a = max |v|, rounded to even.  It is taken as v * (127 / a); a product so near a half that
// its two roundings could have moved it is divided anew (half of the largest value is exactly 63.5, and
// rows of f16 hold such values), so that ties of f16 rows are ties.  For the norm, v = (s * w) * rstd and rounding is monotone,
// so max |v| = max |s * w| * rstd exactly: the sum of squares and the maximum go through one
// reduction, and the row's values are not touched again until they are written.  Maxima are taken
// over the bits of |v| as whole numbers, in which infinities and NaN come out largest.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace p2p {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr float kTiny = 0x1p-100f;  // a row below it counts as zeros (127 / a stays finite)

// 16 bytes of a row: V values.
template <class T>
struct Piece {
  static constexpr int V = 16 / sizeof(T);
  T e[V];
};

// Values [0, n) of the V at p, the others 0.  Whole pieces in one load where rows are aligned.
template <class T, int V>
__device__ __forceinline__ void load_piece(const T* p, int n, bool wide, float (&v)[V]) {
  union {
    uint4 u;
    T e[V];
  } w;
  if (wide && n >= V) {
    w.u = *reinterpret_cast<const uint4*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) w.e[i] = i < n ? p[i] : from_f32<T>(0.f);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = to_f32(w.e[i]);
}

template <class T, int V>
__device__ __forceinline__ void store_piece(T* p, int n, bool wide, const float (&v)[V]) {
  union {
    uint4 u;
    T e[V];
  } w;
#pragma unroll
  for (int i = 0; i < V; ++i) w.e[i] = from_f32<T>(v[i]);
  if (wide && n >= V) {
    *reinterpret_cast<uint4*>(p) = w.u;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = w.e[i];
  }
}

// What a row's values are multiplied with, and its scale.  inv 0: all codes are 0.
struct RowScale {
  float rstd, top, inv, scale;
};

// Adding 1.5 * 2^23 rounds to a whole number, whose low byte is the code.
template <int V>
__device__ __forceinline__ void store_codes(int8_t* p, int n, const float (&v)[V],
                                            const RowScale& sc) {
  constexpr float kRound = 12582912.f;
  float t[V];
  bool near = false;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float c = v[i] * sc.inv;
    t[i] = __fadd_rn(c, kRound);
    near |= fabsf(__fsub_rn(c, __fsub_rn(t[i], kRound))) > 0.49996f;  // 127 * 2^-22 from a half
  }
  if (near) {
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = __fadd_rn(__fdiv_rn(__fmul_rn(v[i], 127.f), sc.top), kRound);
  }
  uint32_t u[V / 4];
#pragma unroll
  for (int i = 0; i < V / 4; ++i) {
    const uint32_t lo = __byte_perm(__float_as_uint(t[4 * i]), __float_as_uint(t[4 * i + 1]), 0x0040),
                   hi = __byte_perm(__float_as_uint(t[4 * i + 2]), __float_as_uint(t[4 * i + 3]), 0x0040);
    u[i] = sc.inv == 0.f ? 0u : __byte_perm(lo, hi, 0x5410);
  }
  if (n >= V) {
    if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
    else *reinterpret_cast<uint32_t*>(p) = u[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = int8_t(u[i / 4] >> (8 * (i % 4)));
  }
}

struct RowSums {
  uint32_t top;  // bits of the largest |value|
  float ss;
};

// The sums of the threads of a row: `warps` consecutive warps of the block, `first` the row's first.
__device__ __forceinline__ RowSums row_reduce(RowSums r, int warps, int first, int warp, int lane,
                                              RowSums* part) {
  r.top = __reduce_max_sync(0xffffffffu, r.top);
#pragma unroll
  for (int o = 16; o; o >>= 1) r.ss += __shfl_xor_sync(0xffffffffu, r.ss, o);
  if (warps == 1) return r;
  if (lane == 0) part[warp] = r;
  asm volatile("bar.sync %0, %1;" ::"r"(1 + first), "r"(32 * warps) : "memory");
  r = part[first];
  for (int i = 1; i < warps; ++i) {
    r.top = max(r.top, part[first + i].top);
    r.ss += part[first + i].ss;
  }
  return r;
}

template <bool NORM>
__device__ __forceinline__ RowScale row_scale(RowSums r, int cols, float eps) {
  RowScale s;
  const float nan = __uint_as_float(0x7fffffffu);
  s.rstd = 1.f;
  if constexpr (NORM)
    s.rstd = r.ss <= 3.4028235e38f
                 ? __fdiv_rn(1.f, __fsqrt_rn(__fdiv_rn(r.ss, float(cols)) + eps))
                 : nan;
  const float a = s.top = __uint_as_float(r.top) * s.rstd;
  if (a < kTiny) {
    s.inv = s.scale = 0.f;
  } else if (a <= 3.4028235e38f) {
    s.inv = __fdiv_rn(127.f, a);
    s.scale = __fdiv_rn(a, 127.f);
  } else {
    s.inv = 0.f;
    s.scale = nan;
  }
  return s;
}

// A row in the registers of `warps` warps, NP pieces a lane.
template <class T, int NP, bool NORM>
__global__ void __launch_bounds__(kThreads)
    rows_kernel(const __grid_constant__ RowsQ8Args a, int warps, int wide) {
  constexpr int V = Piece<T>::V;
  __shared__ RowSums part[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = warp / warps * warps;
  const int64_t row = int64_t(blockIdx.x) * (kWarps / warps) + warp / warps;
  grid_dependency_wait();
  launch_dependents();
  if (row >= a.out.rows) return;
  const int cols = a.out.cols, step = warps * 32 * V;
  const int col0 = ((warp - first) * 32 + lane) * V;
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  float v[NP][V];
#pragma unroll
  for (int i = 0; i < NP; ++i)
    load_piece<T, V>(x + col0 + i * step, cols - (col0 + i * step), wide, v[i]);
  RowSums sums{0u, 0.f};
  if constexpr (NORM) {
    if (a.r) {
      const T* r = static_cast<const T*>(a.r) + row * a.ld_r;
      float u[NP][V];
#pragma unroll
      for (int i = 0; i < NP; ++i)
        load_piece<T, V>(r + col0 + i * step, cols - (col0 + i * step), wide, u[i]);
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] = round_st<T>(v[i][j] + u[i][j]);
    }
    if (a.sum) {
      T* s = static_cast<T*>(a.sum) + row * a.ld_sum;
#pragma unroll
      for (int i = 0; i < NP; ++i)
        store_piece<T, V>(s + col0 + i * step, cols - (col0 + i * step), wide, v[i]);
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = col0 + i * step + j;
        sums.ss += v[i][j] * v[i][j];
        if (a.w) v[i][j] *= c < cols ? __half2float(a.w[c]) : 0.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j)
      sums.top = max(sums.top, __float_as_uint(v[i][j]) & 0x7fffffffu);
  sums = row_reduce(sums, warps, first, warp, lane, part);
  const RowScale sc = row_scale<NORM>(sums, cols, a.eps);
  if constexpr (NORM) {
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] *= sc.rstd;
    if (a.y) {
      T* y = static_cast<T*>(a.y) + row * a.ld_y;
#pragma unroll
      for (int i = 0; i < NP; ++i)
        store_piece<T, V>(y + col0 + i * step, cols - (col0 + i * step), wide, v[i]);
    }
    if (!a.out.q) return;
  }
  int8_t* q = a.out.q + row * a.out.ld;
#pragma unroll
  for (int i = 0; i < NP; ++i)
    store_codes<V>(q + col0 + i * step, cols - (col0 + i * step), v[i], sc);
  if (warp == first && lane == 0) a.out.scale[row] = sc.scale;
}

// Rows too long for the registers of a block: read twice, a block a row.  The second reading takes
// s from where the first one stored it (sum may be x or r).
template <class T, bool NORM>
__global__ void __launch_bounds__(kThreads)
    long_rows_kernel(const __grid_constant__ RowsQ8Args a, int wide) {
  constexpr int V = Piece<T>::V;
  __shared__ RowSums part[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x;
  const int cols = a.out.cols;
  grid_dependency_wait();
  launch_dependents();
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  const T* r = NORM && a.r ? static_cast<const T*>(a.r) + row * a.ld_r : nullptr;
  T* s = NORM && a.sum ? static_cast<T*>(a.sum) + row * a.ld_sum : nullptr;
  RowSums sums{0u, 0.f};
  for (int c = threadIdx.x * V; c < cols; c += kThreads * V) {
    float v[V], u[V];
    load_piece<T, V>(x + c, cols - c, wide, v);
    if (r) {
      load_piece<T, V>(r + c, cols - c, wide, u);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = round_st<T>(v[j] + u[j]);
    }
    if (s) store_piece<T, V>(s + c, cols - c, wide, v);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (NORM) {
        sums.ss += v[j] * v[j];
        if (a.w) v[j] *= c + j < cols ? __half2float(a.w[c + j]) : 0.f;
      }
      sums.top = max(sums.top, __float_as_uint(v[j]) & 0x7fffffffu);
    }
  }
  sums = row_reduce(sums, kWarps, 0, warp, lane, part);
  const RowScale sc = row_scale<NORM>(sums, cols, a.eps);
  T* y = NORM && a.y ? static_cast<T*>(a.y) + row * a.ld_y : nullptr;
  int8_t* q = a.out.q ? a.out.q + row * a.out.ld : nullptr;
  for (int c = threadIdx.x * V; c < cols; c += kThreads * V) {
    float v[V], u[V];
    load_piece<T, V>(s ? s + c : x + c, cols - c, wide, v);
    if (r && !s) {
      load_piece<T, V>(r + c, cols - c, wide, u);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = round_st<T>(v[j] + u[j]);
    }
    if constexpr (NORM) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (a.w) v[j] *= c + j < cols ? __half2float(a.w[c + j]) : 0.f;
        v[j] *= sc.rstd;
      }
    }
    if (y) store_piece<T, V>(y + c, cols - c, wide, v);
    if (q) store_codes<V>(q + c, cols - c, v, sc);
  }
  if (q && threadIdx.x == 0) a.out.scale[row] = sc.scale;
}

// Codes back to values: a warp takes up to kReadPieces pieces a lane of one row.
constexpr int kReadPieces = 4;
template <class T>
__global__ void __launch_bounds__(kThreads)
    read_kernel(const __grid_constant__ ReadQ8Args a, int segments, int wide) {
  constexpr int V = Piece<T>::V;
  const int lane = threadIdx.x & 31;
  const int64_t unit = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  grid_dependency_wait();
  launch_dependents();
  const int64_t i = unit / segments;
  if (i >= a.rows) return;
  const int col0 = (int(unit - i * segments) * kReadPieces * 32 + lane) * V;
  const int64_t row = a.index ? a.index[i] : i;
  const bool inside = row >= 0 && row < a.src.rows;
  if (!inside && row != -1 && lane == 0) atomicOr(a.err, kErrIndex);
  const float scale = inside ? a.src.scale[row] : 0.f;
  const int8_t* q = a.src.q + (inside ? row : 0) * a.src.ld;
  T* out = static_cast<T*>(a.out) + i * a.ld_out;
  union {
    uint32_t u[V / 4];
    int8_t e[V];
  } w[kReadPieces];
#pragma unroll
  for (int p = 0; p < kReadPieces; ++p) {
    const int c = col0 + p * 32 * V, n = a.src.cols - c;
#pragma unroll
    for (int j = 0; j < V / 4; ++j) w[p].u[j] = 0;
    if (!inside) continue;
    if (n >= V) {
      if constexpr (V == 8) {
        const uint2 u = *reinterpret_cast<const uint2*>(q + c);
        w[p].u[0] = u.x;
        w[p].u[1] = u.y;
      } else {
        w[p].u[0] = *reinterpret_cast<const uint32_t*>(q + c);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < n) w[p].e[j] = q[c + j];
    }
  }
#pragma unroll
  for (int p = 0; p < kReadPieces; ++p) {
    const int c = col0 + p * 32 * V, n = a.src.cols - c;
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = inside ? (float(w[p].e[j]) * scale) * a.factor : 0.f;
    if (n > 0) store_piece<T, V>(out + c, n, wide, v);
  }
}

bool on16(const void* p, int64_t pitch_bytes, int64_t rows) {
  return !p || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && (rows == 1 || pitch_bytes % 16 == 0));
}

cudaError_t launch(const void* fn, int64_t blocks, void** args, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelExC(&cfg, fn, args);
}

template <class T, bool NORM>
cudaError_t launch_rows_t(const RowsQ8Args& args, int num_sms, cudaStream_t s) {
  constexpr int V = Piece<T>::V, kMost = 32 / V;  // 32 values a lane
  RowsQ8Args a = args;
  const int64_t es = sizeof(T), rows = a.out.rows;
  int wide = on16(a.x, a.ld_x * es, rows) && on16(a.r, a.ld_r * es, rows) &&
             on16(a.sum, a.ld_sum * es, rows) && on16(a.y, a.ld_y * es, rows);
  const int passes = (a.out.cols + 32 * V - 1) / (32 * V);  // pieces of one warp's lanes
  if (passes > kWarps * kMost) {
    void* p[] = {&a, &wide};
    return launch(reinterpret_cast<const void*>(&long_rows_kernel<T, NORM>), rows, p, s);
  }
  int warps = 1;
  while (warps < kWarps && (passes > warps * kMost ||
                            (passes > warps && rows * warps < int64_t(num_sms) * 32)))
    warps *= 2;
  const int np = (passes + warps - 1) / warps;
  const int64_t blocks = (rows + kWarps / warps - 1) / (kWarps / warps);
  void* p[] = {&a, &warps, &wide};
  const void* fn = np <= 1   ? reinterpret_cast<const void*>(&rows_kernel<T, 1, NORM>)
                   : np <= 2 ? reinterpret_cast<const void*>(&rows_kernel<T, 2, NORM>)
                   : np <= 4 ? reinterpret_cast<const void*>(&rows_kernel<T, 4, NORM>)
                             : reinterpret_cast<const void*>(&rows_kernel<T, kMost, NORM>);
  return launch(fn, blocks, p, s);
}

}  // namespace

cudaError_t launch_rows_q8(const RowsQ8Args& a, int dtype, int num_sms, cudaStream_t s) {
  if (dtype == 0)
    return a.norm ? launch_rows_t<__half, true>(a, num_sms, s)
                  : launch_rows_t<__half, false>(a, num_sms, s);
  return a.norm ? launch_rows_t<float, true>(a, num_sms, s)
                : launch_rows_t<float, false>(a, num_sms, s);
}

cudaError_t launch_read_q8(const ReadQ8Args& args, int dtype, cudaStream_t s) {
  ReadQ8Args a = args;
  const int es = dtype == 0 ? 2 : 4, per = kReadPieces * 32 * (16 / es);
  int segments = (a.src.cols + per - 1) / per;
  int wide = on16(a.out, a.ld_out * es, a.rows);
  const int64_t blocks = (a.rows * segments + kWarps - 1) / kWarps;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  void* p[] = {&a, &segments, &wide};
  return launch(dtype == 0 ? reinterpret_cast<const void*>(&read_kernel<__half>)
                           : reinterpret_cast<const void*>(&read_kernel<float>),
                blocks, p, s);
}

}  // namespace p2p
