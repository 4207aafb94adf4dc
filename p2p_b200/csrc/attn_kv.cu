// attn_kv.cu -- attention of ragged rows over a KV cache of any layout, and of single tokens over
// a 4-bit cache (ATTN, src/scripts/lfm-engine/kernels.js:268-319, on caches that shader has not).
//
// The plain form: one warp per (row, q head), each lane the keys lane, lane + 32, ... with an
// online softmax of its own, joined across lanes at the end.  Every key is read once per row and
// q head.
#include "common.cuh"
#include "kernels.h"
#include "kv_view.cuh"

namespace p2p {
namespace {

constexpr int kWarps = 4;
constexpr float kNegBig = -1e30f;

// The 64 values of kv head kh in cache row `at` of pool k or v.
template <int KVF>
__device__ __forceinline__ void load_head(const KvView& c, bool is_k, int64_t at, int kh,
                                          float (&v)[64]) {
  const unsigned char* base = (is_k ? c.k : c.v) + at * c.row_bytes;
  if constexpr (KVF == kKvF16) {
    const __half* p = reinterpret_cast<const __half*>(base) + kh * 64;
#pragma unroll
    for (int i = 0; i < 64; i += 8) {
      float t[8];
      load8_stream(p + i, t);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[i + k] = t[k];
    }
  } else if constexpr (KVF == kKvI8) {
    const int8_t* p = reinterpret_cast<const int8_t*>(base) + kh * 64;
    const float* sc = is_k ? c.k_scale : c.v_scale;
#pragma unroll
    for (int i = 0; i < 64; ++i)
      v[i] = __fmul_rn(float(p[i]), c.per_channel ? sc[kh * 64 + i] : sc[0]);
  } else {
    const uint32_t* unit = reinterpret_cast<const uint32_t*>(base + kh * kQ4UnitBytes);
    float sc, lo;
    q4_unpack(unit[8], sc, lo);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      float t[8];
      q4_values(unit[w], sc, lo, t);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[8 * w + k] = t[k];
    }
  }
}

template <int KVF>
__global__ void __launch_bounds__(kWarps * 32)
    attn_rows_kernel(const __grid_constant__ AttnKvArgs a) {
  __shared__ float q_s[kWarps][64];
  __shared__ float new_s[kWarps][2][64];
  __shared__ uint32_t unit_s[kWarps][2][9];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t item = int64_t(blockIdx.x) * kWarps + warp;
  const int64_t row = item / a.hq;
  const int h = int(item - row * a.hq), kh = h / (a.hq / a.kv.hkv);
  if (row >= a.at.n_rows) return;
  const int seq = a.at.row_start ? warp_find_seq(a.at.row_start, a.at.nseq, row) : int(row);
  if (seq < 0) return;
  const SeqSpan span = seq_span(a.kv, a.at, seq);
  if (!span.ok) {
    if (lane == 0) atomicOr(a.err, kErrPosBeyondCache);
    return;
  }
  const int pos = span.past + int(row - span.row0);
  const __half* qrow = a.q + row * a.ld_q;
  float q0 = __half2float(qrow[h * 64 + lane]), q1 = __half2float(qrow[h * 64 + 32 + lane]);
  int64_t new_at = 0;
  if (a.fused) {
    const float cs = __half2float(a.rope[int64_t(pos) * 64 + lane]);
    const float sn = __half2float(a.rope[int64_t(pos) * 64 + 32 + lane]);
    float r0, r1;
    norm_rope_head(q0, q1, a.norm_w, a.norm_w != nullptr, a.eps, cs, sn, r0, r1);
    q0 = round_st<__half>(r0);
    q1 = round_st<__half>(r1);
    const __half* kn = qrow + (a.hq + kh) * 64;
    norm_rope_head(__half2float(kn[lane]), __half2float(kn[lane + 32]),
                   a.norm_w ? a.norm_w + 64 : nullptr, a.norm_w != nullptr, a.eps, cs, sn, r0, r1);
    const __half* vn = qrow + (a.hq + a.kv.hkv + kh) * 64;
    new_s[warp][0][lane] = round_st<__half>(r0);
    new_s[warp][0][lane + 32] = round_st<__half>(r1);
    new_s[warp][1][lane] = __half2float(vn[lane]);
    new_s[warp][1][lane + 32] = __half2float(vn[lane + 32]);
    __syncwarp();
    float x[8];  // lanes 0-7: k's unit, 8-15: v's
    const int s = lane & 7, kv = (lane >> 3) & 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = new_s[warp][kv][4 * s + i];
      x[4 + i] = new_s[warp][kv][32 + 4 * s + i];
    }
    q4_store_unit(x, unit_s[warp][kv], lane < 16);
    __syncwarp();
    new_at = kv_row(a.kv, seq, pos);
    if (new_at < 0) {
      if (lane == 0) atomicOr(a.err, kErrPosBeyondCache);
      return;
    }
    if (h % (a.hq / a.kv.hkv) == 0 && lane < 18) {
      unsigned char* dst = (lane < 9 ? a.kv.k : a.kv.v) + new_at * a.kv.row_bytes +
                           kh * kQ4UnitBytes;
      reinterpret_cast<uint32_t*>(dst)[lane % 9] = unit_s[warp][lane / 9][lane % 9];
    }
  }
  q_s[warp][lane] = q0;
  q_s[warp][lane + 32] = q1;
  __syncwarp();
  float m = kNegBig, l = 0.f, acc[64];
#pragma unroll
  for (int i = 0; i < 64; ++i) acc[i] = 0.f;
  bool bad = false;
  for (int j = lane; j <= pos; j += 32) {
    const bool is_new = a.fused && j == pos;
    const int64_t at = is_new ? 0 : kv_row(a.kv, seq, j);
    if (at < 0) {
      bad = true;
      continue;
    }
    float v[64];
    if (is_new) {
      KvView c = a.kv;  // the unit in shared memory
      c.k = reinterpret_cast<unsigned char*>(unit_s[warp][0]);
      load_head<KVF>(c, true, 0, 0, v);
    } else {
      load_head<KVF>(a.kv, true, at, kh, v);
    }
    float sc = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) sc = fmaf(q_s[warp][i], v[i], sc);
    sc *= a.scale_log2;
    const float mn = fmaxf(m, sc), c = exp2f(m - mn), p = exp2f(sc - mn);
    m = mn;
    l = fmaf(l, c, p);
    if (is_new) {
      KvView cv = a.kv;
      cv.v = reinterpret_cast<unsigned char*>(unit_s[warp][1]);
      load_head<KVF>(cv, false, 0, 0, v);
    } else {
      load_head<KVF>(a.kv, false, at, kh, v);
    }
#pragma unroll
    for (int i = 0; i < 64; ++i) acc[i] = fmaf(acc[i], c, p * v[i]);
  }
  if (__any_sync(0xffffffffu, bad)) {
    if (lane == 0) atomicOr(a.err, kErrPosBeyondCache);
    return;
  }
  float mx = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float c = exp2f(m - mx);
  l *= c;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  __half* dst = a.out + row * a.ld_o + h * 64;
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    float t = acc[i] * c;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) dst[i] = __float2half_rn(t / l);
  }
}

}  // namespace

cudaError_t launch_attn_kv(const AttnKvArgs& a, cudaStream_t s) {
  const int64_t blocks = (a.at.n_rows * a.hq + kWarps - 1) / kWarps;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  const dim3 g{unsigned(blocks)};
  if (a.kv.format == kKvF16) attn_rows_kernel<kKvF16><<<g, kWarps * 32, 0, s>>>(a);
  else if (a.kv.format == kKvI8) attn_rows_kernel<kKvI8><<<g, kWarps * 32, 0, s>>>(a);
  else attn_rows_kernel<kKvQ4><<<g, kWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace p2p
