// rows_q8.cu -- rows of 8-bit integers with a scale each: made from f16 / f32 rows, alone or behind
// the residual addition and RMS norm of a decoder layer (ADD_RMS,
// src/scripts/lfm-engine/kernels.js:146-182), and read back as values (the embedding lookup).
//
// All three move bytes: a row is read once, kept in registers (as it lies in memory, 4 words for 16
// bytes), reduced and written once.  A code is 127 v / a, a = max |v|, rounded to even, taken as
// v * (127 / a) + 1.5 * 2^23 in one operation.  Of f16 rows ties are exact: with 127 / a rounded up, half
// of the largest value (63.5 exactly) goes to 64, no other quotient lies so near a half that the factor's
// last place could move it ((c + 1/2) 2^-18 at least, against (c + 1/2) 2^-23), and rows whose a has a
// multiple of 127 for its 11 bits, which alone give other ties, are divided value by value.  For the norm,
// v = (s * w) * rstd and rounding is monotone, so max |v| = max |s * w| * rstd exactly: the sum of squares
// and the maximum go through one reduction.
//   A row is in the hands of as few warps as hold it, 4 pieces of 16 bytes a lane: what a warp does once
// for a row costs as much as 20 to 40 of its values (65536 rows of 1024 f16 values in 36 us by warps, 68
// by pairs of warps, 131 by eight; blocks that walk rows, with or without the next row on its way, were
// slower: 39 to 43).
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace p2p {
namespace {

constexpr int kThreads = 256;         // of a block whose warps take a row each
constexpr int kWarps = kThreads / 32;
constexpr int kMostWarps = 16;        // of a row
constexpr int kMostPieces = 4;        // of a lane
constexpr float kTiny = 0x1p-100f;  // a row below it counts as zeros (127 / a stays finite)

// max(|a|, |b|, |c|), NaN if one of them is.
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 16 bytes of a row as they lie in memory: V values.
template <class T>
union Piece {
  static constexpr int V = 16 / sizeof(T);
  uint4 u;
  T e[V];
  __half2 h[4];
  __device__ __forceinline__ Pair get(int i) const {  // values 2i and 2i + 1
    if constexpr (sizeof(T) == 2) {
      const float2 f = __half22float2(h[i]);
      return pair(f.x, f.y);
    } else {
      return pair(e[2 * i], e[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void set(int i, Pair p) {
    if constexpr (sizeof(T) == 2) {
      h[i] = __floats2half2_rn(p.f[0], p.f[1]);
    } else {
      e[2 * i] = p.f[0];
      e[2 * i + 1] = p.f[1];
    }
  }
};

// The columns of a row over the threads that hold it: a thread's piece is V neighbours, whatever the
// rows' alignment (so that sums, and with them all results, do not depend on it).
template <int V>
struct Columns {
  int first, threads, cols;  // the thread's place among those of the row
  __device__ __forceinline__ int at(int piece, int e = 0) const {
    return (piece * threads + first) * V + e;
  }
  __device__ __forceinline__ bool whole(int piece) const { return at(piece, V - 1) < cols; }
};

// Rows that start on 16-byte boundaries (WIDE) are read and written piece by piece.  Others go value by
// value, neighbours in neighbouring lanes, so that each access of a warp is still one contiguous stretch,
// and change hands through a warp's 512 bytes of shared memory (`turn`).  Value j of lane l is then the
// warp's value 32 j + l.
template <bool WIDE, class T>
__device__ __forceinline__ void load_piece(Piece<T>& w, const T* row, const Columns<Piece<T>::V>& c,
                                           int piece) {
  constexpr int V = Piece<T>::V;
  const int lane = threadIdx.x & 31, col = c.at(piece) - lane * V + lane;
  if (WIDE && c.whole(piece)) {
    w.u = *reinterpret_cast<const uint4*>(row + c.at(piece));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int at = WIDE ? c.at(piece, j) : col + 32 * j;
      w.e[j] = at < c.cols ? row[at] : from_f32<T>(0.f);
    }
  }
}
// A loaded piece's values to the threads they belong to.
template <bool WIDE, class T>
__device__ __forceinline__ void turn_loaded(Piece<T>& w, uint4* turn) {
  if constexpr (!WIDE) {
    const int lane = threadIdx.x & 31;
    T* t = reinterpret_cast<T*>(turn);
#pragma unroll
    for (int j = 0; j < Piece<T>::V; ++j) t[32 * j + lane] = w.e[j];
    __syncwarp();
    w.u = turn[lane];
    __syncwarp();
  }
}
template <bool WIDE, class T>
__device__ __forceinline__ void store_piece(const Piece<T>& w, T* row, const Columns<Piece<T>::V>& c,
                                            int piece, uint4* turn) {
  constexpr int V = Piece<T>::V;
  const int lane = threadIdx.x & 31;
  if constexpr (WIDE) {
    if (c.whole(piece)) {
      *reinterpret_cast<uint4*>(row + c.at(piece)) = w.u;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c.at(piece, j) < c.cols) row[c.at(piece, j)] = w.e[j];
    }
  } else {
    const int col = c.at(piece) - lane * V + lane;
    const T* t = reinterpret_cast<const T*>(turn);
    turn[lane] = w.u;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (col + 32 * j < c.cols) row[col + 32 * j] = t[32 * j + lane];
    __syncwarp();
  }
}
// The V norm weights of a piece (0 behind the row's end; ones without weights).
template <bool WIDE, int V>
__device__ __forceinline__ void load_weights(__half2 (&w)[V / 2], const __half* row,
                                             const Columns<V>& c, int piece) {
  union {
    uint4 u4;
    uint2 u2;
    __half e[V];
    __half2 h[V / 2];
  } x;
  if (!row) {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) x.h[j] = __float2half2_rn(1.f);
  } else if (WIDE && c.whole(piece)) {
    if constexpr (V == 8) x.u4 = *reinterpret_cast<const uint4*>(row + c.at(piece));
    else x.u2 = *reinterpret_cast<const uint2*>(row + c.at(piece));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      x.e[j] = c.at(piece, j) < c.cols ? row[c.at(piece, j)] : __half(0.f);
  }
#pragma unroll
  for (int j = 0; j < V / 2; ++j) w[j] = x.h[j];
}
__device__ __forceinline__ Pair wide2(__half2 h) {
  const float2 f = __half22float2(h);
  return pair(f.x, f.y);
}

// What a row's values are multiplied with, and its scale.  inv 0: all codes are 0.
struct RowScale {
  float rstd, top, inv, scale;
  bool divide;
};

// Adding 1.5 * 2^23 rounds to a whole number, whose low byte is the code.
template <int V>
__device__ __forceinline__ void store_codes(int8_t* row, const Columns<V>& c, int piece,
                                            const Pair (&v)[V / 2], const RowScale& sc) {
  constexpr float kRound = 12582912.f;
  const Pair inv = pair(sc.inv, sc.inv), up = pair(kRound, kRound);
  Pair t[V / 2];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) t[i] = mad2(v[i], inv, up);
  if (sc.divide) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        t[i].f[j] = __fadd_rn(__fdiv_rn(__fmul_rn(v[i].f[j], 127.f), sc.top), kRound);
  }
  uint32_t u[V / 4];
#pragma unroll
  for (int i = 0; i < V / 4; ++i) {
    const uint32_t lo = __byte_perm(__float_as_uint(t[2 * i].f[0]), __float_as_uint(t[2 * i].f[1]),
                                    0x0040),
                   hi = __byte_perm(__float_as_uint(t[2 * i + 1].f[0]),
                                    __float_as_uint(t[2 * i + 1].f[1]), 0x0040);
    u[i] = sc.inv == 0.f ? 0u : __byte_perm(lo, hi, 0x5410);
  }
  if (c.whole(piece)) {
    int8_t* p = row + c.at(piece);
    if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
    else *reinterpret_cast<uint32_t*>(p) = u[0];
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (c.at(piece, j) < c.cols) row[c.at(piece, j)] = int8_t(u[j / 4] >> (8 * (j % 4)));
  }
}

struct RowSums {
  float top, ss;  // the largest |value|, the sum of squares
};

// The sums of the threads of a row: a warp, or the `warps` of the block.
template <bool NORM>
__device__ __forceinline__ RowSums row_reduce(RowSums r, int warps, int warp, int lane,
                                              RowSums* part) {
  // as whole numbers, infinities and NaN come out largest
  r.top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(r.top)));
  if constexpr (NORM) {
#pragma unroll
    for (int o = 16; o; o >>= 1) r.ss += __shfl_xor_sync(0xffffffffu, r.ss, o);
  }
  if (warps == 1) return r;
  if (lane == 0) part[warp] = r;
  __syncthreads();
  r = lane < warps ? part[lane] : RowSums{0.f, 0.f};
  r.top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(r.top)));
  if constexpr (NORM) {
#pragma unroll
    for (int o = kMostWarps / 2; o; o >>= 1) r.ss += __shfl_xor_sync(0xffffffffu, r.ss, o);
    r.ss = __shfl_sync(0xffffffffu, r.ss, 0);
  }
  return r;
}

// Every operation rounded.  (With approximations of 2^-22 for the norm's root and quotients 8192 rows of 2048
// f16 values take 21.7 us instead of 22.4, and an f32 y and the scales are up to four units in the last place
// off.)
template <bool NORM, bool F16>
__device__ __forceinline__ RowScale row_scale(RowSums r, int cols, float eps) {
  constexpr bool kTies = F16 && !NORM;
  RowScale s;
  const float nan = __uint_as_float(0x7fffffffu);
  s.rstd = 1.f;
  if constexpr (NORM)
    s.rstd = r.ss <= 3.4028235e38f
                 ? __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(__fdiv_rn(r.ss, float(cols)), eps)))
                 : nan;
  const float a = s.top = r.top * s.rstd;
  if (a < kTiny) {
    s.inv = s.scale = 0.f;
  } else if (a <= 3.4028235e38f) {
    s.inv = kTies ? __fdiv_ru(127.f, a) : __fdiv_rn(127.f, a);
    s.scale = __fdiv_rn(a, 127.f);
  } else {
    s.inv = 0.f;
    s.scale = nan;
  }
  s.divide = kTies && (((__float_as_uint(a) >> 13) & 0x3ff) | 0x400) % 127 == 0;
  return s;
}

// s = x + r as it is stored.  (Two f16 values add up to the same f16 value in one rounding and through
// f32: what a f32 sum drops lies below half of the f16 sum's last place, and never on it.)
template <class T>
__device__ __forceinline__ void add_piece(Piece<T>& x, const Piece<T>& r) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x.h[j] = __hadd2(x.h[j], r.h[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j) x.set(j, add2(x.get(j), r.get(j)));
  }
}

// A piece's part of the row's sums.
template <bool NORM, bool WIDE, class T>
__device__ __forceinline__ void sum_piece(RowSums& sums, Pair& ss, const Piece<T>& x,
                                          const RowsQ8Args& a,
                                          const Columns<Piece<T>::V>& c, int piece) {
  constexpr int V = Piece<T>::V;
  if constexpr (!NORM && sizeof(T) == 2) {
    const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(x.h[0]), __habs2(x.h[1])),
                                  __hmax2_nan(__habs2(x.h[2]), __habs2(x.h[3])));
    sums.top = max_abs3(sums.top, __low2float(m), __high2float(m));
  } else {
    __half2 w[V / 2];
    if constexpr (NORM) load_weights<WIDE, V>(w, a.w, c, piece);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      Pair v = x.get(j);
      if constexpr (NORM) {
        ss = mad2(v, v, ss);
        v = mul2(v, wide2(w[j]));
      }
      sums.top = max_abs3(sums.top, v.f[0], v.f[1]);
    }
  }
}
// A piece of what the call stores behind the reduction.
template <bool NORM, bool WIDE, class T>
__device__ __forceinline__ void finish_piece(const Piece<T>& x, const RowScale& sc,
                                             const RowsQ8Args& a, int64_t row,
                                             const Columns<Piece<T>::V>& c, int piece,
                                             uint4* turn) {
  constexpr int V = Piece<T>::V;
  Pair v[V / 2];
  __half2 w[V / 2];
  if constexpr (NORM) load_weights<WIDE, V>(w, a.w, c, piece);
#pragma unroll
  for (int j = 0; j < V / 2; ++j) {
    v[j] = x.get(j);
    if constexpr (NORM) v[j] = mul2(mul2(v[j], wide2(w[j])), pair(sc.rstd, sc.rstd));
  }
  if constexpr (NORM) {
    if (a.y) {
      Piece<T> y;
#pragma unroll
      for (int j = 0; j < V / 2; ++j) y.set(j, v[j]);
      store_piece<WIDE>(y, static_cast<T*>(a.y) + row * a.ld_y, c, piece, turn);
    }
    if (!a.out.q) return;
  }
  store_codes<V>(a.out.q + row * a.out.ld, c, piece, v, sc);
}

// The words of a piece as they are: what was computed from them before is not kept beside them.
template <class T>
__device__ __forceinline__ void keep_words(Piece<T>& x) {
  asm volatile("" : "+r"(x.u.x), "+r"(x.u.y), "+r"(x.u.z), "+r"(x.u.w));
}

// A row in the registers of a warp (warps 1: a row a warp) or of a block of `warps` warps, NP pieces a
// lane.
template <class T, int NP, bool NORM, bool WIDE>
__global__ void __launch_bounds__(32 * kMostWarps, NP <= 4 ? 3 : 1)
    rows_kernel(const __grid_constant__ RowsQ8Args a, int warps) {
  __shared__ RowSums part[kMostWarps];
  __shared__ uint4 turns[WIDE ? 1 : kMostWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = warps == 1 ? int64_t(blockIdx.x) * kWarps + warp : blockIdx.x;
  const int part_of = warps == 1 ? 0 : warp;
  grid_dependency_wait();
  launch_dependents();
  if (row >= a.out.rows) return;
  const Columns<Piece<T>::V> c{part_of * 32 + lane, warps * 32, a.out.cols};
  uint4* turn = turns[WIDE ? 0 : warp];
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  Piece<T> v[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) load_piece<WIDE>(v[i], x, c, i);
  if constexpr (NORM) {
    if (a.r) {  // added as the two were loaded
      const T* r = static_cast<const T*>(a.r) + row * a.ld_r;
      Piece<T> u[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) load_piece<WIDE>(u[i], r, c, i);
#pragma unroll
      for (int i = 0; i < NP; ++i) add_piece(v[i], u[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < NP; ++i) turn_loaded<WIDE>(v[i], turn);
  if constexpr (NORM) {
    if (a.sum) {
      T* s = static_cast<T*>(a.sum) + row * a.ld_sum;
#pragma unroll
      for (int i = 0; i < NP; ++i) store_piece<WIDE>(v[i], s, c, i, turn);
    }
  }
  RowSums sums{0.f, 0.f};
  Pair ss = pair(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < NP; ++i) sum_piece<NORM, WIDE>(sums, ss, v[i], a, c, i);
  sums.ss = ss.f[0] + ss.f[1];
  sums = row_reduce<NORM>(sums, warps, warp, lane, part);
#pragma unroll
  for (int i = 0; i < NP; ++i) keep_words(v[i]);
  const RowScale sc = row_scale<NORM, sizeof(T) == 2>(sums, c.cols, a.eps);
#pragma unroll
  for (int i = 0; i < NP; ++i) finish_piece<NORM, WIDE>(v[i], sc, a, row, c, i, turn);
  if (a.out.q && part_of == 0 && lane == 0) a.out.scale[row] = sc.scale;
}

// Rows too long for the registers of a block: read twice, a block a row.  The second reading takes
// s from where the first one stored it (sum may be x or r).
template <class T, bool NORM, bool WIDE>
__global__ void __launch_bounds__(kThreads)
    long_rows_kernel(const __grid_constant__ RowsQ8Args a) {
  __shared__ RowSums part[kWarps];
  __shared__ uint4 turns[WIDE ? 1 : kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x;
  grid_dependency_wait();
  launch_dependents();
  const Columns<Piece<T>::V> c{int(threadIdx.x), kThreads, a.out.cols};
  const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
  const T* r = NORM && a.r ? static_cast<const T*>(a.r) + row * a.ld_r : nullptr;
  T* s = NORM && a.sum ? static_cast<T*>(a.sum) + row * a.ld_sum : nullptr;
  RowSums sums{0.f, 0.f};
  Pair ss = pair(0.f, 0.f);
  uint4* turn = turns[WIDE ? 0 : warp];
  const int pieces = (c.cols + kThreads * Piece<T>::V - 1) / (kThreads * Piece<T>::V);
  for (int i = 0; i < pieces; ++i) {
    Piece<T> v, u;
    load_piece<WIDE>(v, x, c, i);
    if (r) {
      load_piece<WIDE>(u, r, c, i);
      add_piece(v, u);
    }
    turn_loaded<WIDE>(v, turn);
    if (s) store_piece<WIDE>(v, s, c, i, turn);
    sum_piece<NORM, WIDE>(sums, ss, v, a, c, i);
  }
  sums.ss = ss.f[0] + ss.f[1];
  sums = row_reduce<NORM>(sums, kWarps, warp, lane, part);
  const RowScale sc = row_scale<NORM, sizeof(T) == 2>(sums, c.cols, a.eps);
  for (int i = 0; i < pieces; ++i) {
    Piece<T> v, u;
    load_piece<WIDE>(v, s ? s : x, c, i);
    if (r && !s) {
      load_piece<WIDE>(u, r, c, i);
      add_piece(v, u);
    }
    turn_loaded<WIDE>(v, turn);
    finish_piece<NORM, WIDE>(v, sc, a, row, c, i, turn);
  }
  if (a.out.q && threadIdx.x == 0) a.out.scale[row] = sc.scale;
}

// Codes back to values: a warp takes kReadPieces pieces a lane, of a segment of one row, or (SHORT: rows of
// that many pieces, 1 or 2) of several rows (a row a warp: 33933 rows of 320 in 19.8 us, 13.2 so).
constexpr int kReadPieces = 4;
template <class T, bool WIDE, int SHORT>
__global__ void __launch_bounds__(kThreads)
    read_kernel(const __grid_constant__ ReadQ8Args a, int segments) {
  constexpr int V = Piece<T>::V, kRows = SHORT ? kReadPieces / SHORT : 1;
  __shared__ uint4 turns[WIDE ? 1 : kWarps][32];
  const int lane = threadIdx.x & 31;
  const int64_t unit = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  grid_dependency_wait();
  launch_dependents();
  const int64_t first = SHORT ? unit * kRows : unit / segments;
  if (first >= a.rows) return;
  const int piece0 = SHORT ? 0 : int(unit - first * segments) * kReadPieces;
  const Columns<V> c{lane, 32, a.src.cols};
  float scale[kRows];
  const int8_t* q[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t i = first + r;
    const int64_t row = i >= a.rows ? -1 : a.index ? a.index[i] : i;
    const bool inside = row >= 0 && row < a.src.rows;
    if (!inside && row != -1 && lane == 0) atomicOr(a.err, kErrIndex);
    scale[r] = inside ? a.src.scale[row] : 0.f;
    q[r] = inside ? a.src.q + row * a.src.ld : nullptr;
  }
  union {
    uint32_t u[V / 4];
    int8_t e[V];
  } w[kReadPieces];
#pragma unroll
  for (int p = 0; p < kReadPieces; ++p) {
    const int piece = SHORT ? p % (SHORT ? SHORT : 1) : piece0 + p;
    const int8_t* from = q[SHORT ? p / (SHORT ? SHORT : 1) : 0];
#pragma unroll
    for (int j = 0; j < V / 4; ++j) w[p].u[j] = 0;
    if (!from) continue;
    if (c.whole(piece)) {
      if constexpr (V == 8) {
        const uint2 u = *reinterpret_cast<const uint2*>(from + c.at(piece));
        w[p].u[0] = u.x;
        w[p].u[1] = u.y;
      } else {
        w[p].u[0] = *reinterpret_cast<const uint32_t*>(from + c.at(piece));
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c.at(piece, j) < c.cols) w[p].e[j] = from[c.at(piece, j)];
    }
  }
#pragma unroll
  for (int p = 0; p < kReadPieces; ++p) {
    const int r = SHORT ? p / (SHORT ? SHORT : 1) : 0;
    if (first + r >= a.rows) break;
    Piece<T> v;
#pragma unroll
    for (int j = 0; j < V; ++j) v.e[j] = from_f32<T>((float(w[p].e[j]) * scale[r]) * a.factor);
    store_piece<WIDE>(v, static_cast<T*>(a.out) + (first + r) * a.ld_out, c,
                      SHORT ? p % (SHORT ? SHORT : 1) : piece0 + p, turns[WIDE ? 0 : threadIdx.x >> 5]);
  }
}

bool on16(const void* p, int64_t pitch_bytes, int64_t rows) {
  return !p || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && (rows == 1 || pitch_bytes % 16 == 0));
}

cudaError_t launch(const void* fn, int64_t blocks, void** args, cudaStream_t s,
                   int threads = kThreads) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(blocks));
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelExC(&cfg, fn, args);
}

template <class T, bool NORM, bool WIDE>
cudaError_t launch_rows_t(RowsQ8Args a, int num_sms, cudaStream_t s) {
  constexpr int V = Piece<T>::V;
  const int64_t rows = a.out.rows;
  const int passes = (a.out.cols + 32 * V - 1) / (32 * V);  // pieces of one warp's lanes
  if (passes > kMostWarps * kMostPieces) {
    void* p[] = {&a};
    return launch(reinterpret_cast<const void*>(&long_rows_kernel<T, NORM, WIDE>), rows, p, s);
  }
  // As few warps a row as hold it in kMostPieces pieces a lane, the norm, which holds x and the residual,
  // in two (8192 rows of 2048 f16 values 22.4 us, 23.8 in four; 13.6 and 15.2 for 1024), one warp also with
  // eight pieces a lane (65536 rows of 1024 f32 values are quantised in 49 us then, 68 by pairs of warps); but
  // where rows are few, as many as the row has pieces for, up to 8.
  const int most = NORM && passes <= 2 * kMostWarps ? 2 : kMostPieces;
  int warps = 1;
  while (passes > warps * (!NORM && V == 4 && warps == 1 ? 8 : most) ||
         (warps < 8 && passes > warps && rows * warps < int64_t(num_sms) * 32))
    warps *= 2;
  const int np = (passes + warps - 1) / warps;
  const int64_t blocks = warps == 1 ? (rows + kWarps - 1) / kWarps : rows;
  void* p[] = {&a, &warps};
  const void* fn = np <= 1   ? reinterpret_cast<const void*>(&rows_kernel<T, 1, NORM, WIDE>)
                   : np <= 2 ? reinterpret_cast<const void*>(&rows_kernel<T, 2, NORM, WIDE>)
                   : np <= 3 ? reinterpret_cast<const void*>(&rows_kernel<T, 3, NORM, WIDE>)
                   : np <= 4 ? reinterpret_cast<const void*>(&rows_kernel<T, 4, NORM, WIDE>)
                             : reinterpret_cast<const void*>(&rows_kernel<T, NORM || V == 8 ? 4 : 8, NORM, WIDE>);
  return launch(fn, blocks, p, s, warps == 1 ? kThreads : 32 * warps);
}

template <class T>
cudaError_t launch_rows(const RowsQ8Args& a, int num_sms, cudaStream_t s) {
  const int64_t es = sizeof(T), rows = a.out.rows;
  const bool wide = on16(a.x, a.ld_x * es, rows) && on16(a.r, a.ld_r * es, rows) &&
                    on16(a.sum, a.ld_sum * es, rows) && on16(a.y, a.ld_y * es, rows) &&
                    on16(a.w, 0, 1);
  if (a.norm)
    return wide ? launch_rows_t<T, true, true>(a, num_sms, s)
                : launch_rows_t<T, true, false>(a, num_sms, s);
  return wide ? launch_rows_t<T, false, true>(a, num_sms, s)
              : launch_rows_t<T, false, false>(a, num_sms, s);
}

template <class T, bool WIDE>
cudaError_t launch_read(ReadQ8Args a, cudaStream_t s) {
  constexpr int per = 32 * Piece<T>::V;
  const int pieces = (a.src.cols + per - 1) / per;
  int segments = (pieces + kReadPieces - 1) / kReadPieces;
  const int64_t units = pieces <= 2 ? (a.rows * pieces + kReadPieces - 1) / kReadPieces : a.rows * segments;
  const int64_t blocks = (units + kWarps - 1) / kWarps;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  void* p[] = {&a, &segments};
  return launch(pieces == 1   ? reinterpret_cast<const void*>(&read_kernel<T, WIDE, 1>)
                : pieces == 2 ? reinterpret_cast<const void*>(&read_kernel<T, WIDE, 2>)
                              : reinterpret_cast<const void*>(&read_kernel<T, WIDE, 0>),
                blocks, p, s);
}

}  // namespace

cudaError_t launch_rows_q8(const RowsQ8Args& a, int dtype, int num_sms, cudaStream_t s) {
  return dtype == 0 ? launch_rows<__half>(a, num_sms, s) : launch_rows<float>(a, num_sms, s);
}

cudaError_t launch_read_q8(const ReadQ8Args& a, int dtype, cudaStream_t s) {
  const bool wide = on16(a.out, a.ld_out * (dtype == 0 ? 2 : 4), a.rows);
  if (dtype == 0) return wide ? launch_read<__half, true>(a, s) : launch_read<__half, false>(a, s);
  return wide ? launch_read<float, true>(a, s) : launch_read<float, false>(a, s);
}

}  // namespace p2p
