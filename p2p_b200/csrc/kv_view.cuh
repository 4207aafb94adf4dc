// kv_view.cuh -- a KV cache of any layout as the batched operators see it: where a key's row
// lies, whether a sequence fits, and the 4-bit row format.
//
// 4-bit rows: a token's row holds one 36-byte unit per kv head -- eight 32-bit words of codes
// (dim 8w + i is nibble i of word w) and one word of parameters (f16 scale in the low half, f16
// lowest value lo in the high half) -- padded to a multiple of 16 bytes, so that whole rows move
// with 16-byte and bulk copies and a page is one contiguous run.  A value is code * scale + lo.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace p2p {

// The chunk of sequence i: its first row, its rows, its position, and whether all of them lie
// inside the rows, the lengths and the cache (the pages' own numbers are kv_row's to check).
struct SeqSpan {
  int past, row0, len;
  bool ok;
};

__host__ __device__ __forceinline__ bool span_fits(const KvView& c, const ChunkIndex& x, int past,
                                                  int row0, int len, int off) {
  const int64_t end = int64_t(past) + len;
  return past >= 0 && row0 >= 0 && len >= 0 && int64_t(row0) + len <= x.n_rows &&
         end <= x.max_len &&
         (c.table != nullptr ? end <= 0 || ((end - 1) >> c.shift) < c.max_blocks
                             : off >= 0 && int64_t(off) + end <= c.kv_rows);
}
// The same for one token behind `past` keys (no chunk rows to check).
__host__ __device__ __forceinline__ bool one_token_fits(const KvView& c, const ChunkIndex& x,
                                                       int past, int off) {
  return span_fits(c, x, past, 0, 1, off);
}

__host__ __device__ __forceinline__ SeqSpan seq_span(const KvView& c, const ChunkIndex& x, int i) {
  SeqSpan s;
  s.past = x.past[i];
  if (x.row_start != nullptr) {
    s.row0 = x.row_start[i];
    s.len = x.row_start[i + 1] - s.row0;
  } else {  // one row per sequence
    s.row0 = i;
    s.len = 1;
  }
  s.ok = span_fits(c, x, s.past, s.row0, s.len, c.table == nullptr ? c.offsets[i] : 0);
  return s;
}

// Cache row of key `pos` of sequence i (a valid position), or -1 when its page is outside the pool.
__host__ __device__ __forceinline__ int64_t kv_row(const KvView& c, int i, int pos) {
  if (c.table == nullptr) return int64_t(c.offsets[i]) + pos;
  const int32_t pg = c.table[int64_t(i) * c.max_blocks + (pos >> c.shift)];
  if (pg < 0 || int64_t(pg) >= c.kv_rows) return -1;
  return (int64_t(pg) << c.shift) | (pos & ((1 << c.shift) - 1));
}

// The sequence whose chunk holds row r: the number of i in [1, nseq] with row_start[i] <= r, 32
// entries a step.  -1 when no sequence's rows reach r, and whatever row_start holds, a sequence that is
// returned has r among its rows.  count(f): for how many of the 32 lanes f(lane) holds.
template <class Count>
__host__ __device__ __forceinline__ int find_seq(const int32_t* row_start, int nseq, int64_t r,
                                                 Count count) {
  int lo = 0, n = nseq;  // candidates lo .. lo + n - 1; every entry before lo is <= r
  while (n > 32) {
    const int step = (n + 31) / 32;
    const int below = count([&](int lane) {  // the last candidate of the lane's part
      const int end = (lane + 1) * step;
      return row_start[lo + (end < n ? end : n)] <= r;
    });
    if (below == 32) return -1;
    const int skip = below * step < n ? below * step : n;
    lo += skip;
    n = step < n - skip ? step : n - skip;
    if (n <= 0) return -1;
  }
  const int seq =
      lo + count([&](int lane) { return lane < n && row_start[lo + lane + 1] <= r; });
  return seq < nseq && seq < lo + n && row_start[seq] <= r && r < row_start[seq + 1] ? seq : -1;
}
// The same by a whole warp.
__device__ __forceinline__ int warp_find_seq(const int32_t* row_start, int nseq, int64_t r) {
  const int lane = threadIdx.x & 31;
  return find_seq(row_start, nseq, r,
                  [&](auto f) { return __popc(__ballot_sync(0xffffffffu, f(lane))); });
}

// ---- the 4-bit rows ---------------------------------------------------------------------------
__device__ __forceinline__ float q4_scale(float lo, float hi, __half& stored) {
  stored = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.0f));
  return __half2float(stored);
}
__device__ __forceinline__ uint32_t q4_code(float x, float lo, float scale) {
  if (!(scale > 0.f)) return 0u;
  const float q = rintf(__fdiv_rn(__fsub_rn(x, lo), scale));
  return uint32_t(fminf(fmaxf(q, 0.f), 15.f));
}
__device__ __forceinline__ uint32_t q4_params(__half scale, float lo) {
  return uint32_t(__half_as_ushort(scale)) |
         (uint32_t(__half_as_ushort(__float2half_rn(lo))) << 16);
}
__device__ __forceinline__ void q4_unpack(uint32_t params, float& scale, float& lo) {
  scale = __half2float(__ushort_as_half(static_cast<unsigned short>(params & 0xffffu)));
  lo = __half2float(__ushort_as_half(static_cast<unsigned short>(params >> 16)));
}
// The eight values of a code word (the product of a code and an f16 scale is exact in f32).
__device__ __forceinline__ void q4_values(uint32_t w, float scale, float lo, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = fmaf(float((w >> (4 * i)) & 15u), scale, lo);
}

// A head's 64 values held by 8 consecutive lanes (lane s = lane & 7: dims 4s .. 4s+3 in x[0..3],
// 32 + 4s .. 32 + 4s + 3 in x[4..7]) quantised into its unit: lane s stores one code word, lane 0
// the parameters too.  Called by whole warps; lanes with store == false compute but do not store.
__device__ __forceinline__ void q4_store_unit(const float (&x)[8], uint32_t* unit, bool store) {
  const int s = threadIdx.x & 7;
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  __half sh;
  const float sc = q4_scale(lo, hi, sh);
  uint32_t a = 0, b = 0;  // 16 bits each: the codes of x[0..3] and of x[4..7]
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a |= q4_code(x[i], lo, sc) << (4 * i);
    b |= q4_code(x[4 + i], lo, sc) << (4 * i);
  }
  // even lanes store word s / 2 (their a, the next lane's a), odd lanes word 4 + s / 2
  const bool odd = (s & 1) != 0;
  const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
  const uint32_t w = odd ? (got | (b << 16)) : (a | (got << 16));
  if (store) {
    unit[odd ? 4 + (s >> 1) : (s >> 1)] = w;
    if (s == 0) unit[8] = q4_params(sh, lo);
  }
}

}  // namespace p2p
