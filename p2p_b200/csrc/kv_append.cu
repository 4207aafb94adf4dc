// kv_append.cu -- rows of ragged prompt chunks into a KV cache of any layout (QK_PREP,
// src/scripts/lfm-engine/kernels.js:216-266, with the append generalised), cached sequences read
// back, and f16 rows to the 4-bit format.
//
// All three move bytes and compute little.  A unit -- the 64 values of one (row, head) -- belongs
// to 8 lanes, so a warp works on four units and each of its loads and stores covers whole 32-byte
// sectors: lane s of a unit holds dims 4s .. 4s+3 and 32+4s .. 32+4s+3, which are rotate-half
// partners, so the rotation needs no exchange.
#include "common.cuh"
#include "kernels.h"
#include "kv_view.cuh"

namespace p2p {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void load4(const __half* p, float* v) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
  v[0] = a.x;
  v[1] = a.y;
  v[2] = b.x;
  v[3] = b.y;
}
__device__ __forceinline__ void store4(__half* p, const float* v) {
  const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
  uint2 w;
  w.x = *reinterpret_cast<const uint32_t*>(&a);
  w.y = *reinterpret_cast<const uint32_t*>(&b);
  *reinterpret_cast<uint2*>(p) = w;
}

// x (8 values of a unit per lane) normed in place: the sum of squares in the shader's tree order
// (kernels.js:246-251: t[i] = v[i]^2 + v[i+32]^2, then pairs 16, 8, 4, 2, 1 apart, the first three
// of them in the neighbouring lanes), each IEEE operation on its own, so bit-identical to it.
__device__ __forceinline__ void norm_unit(float (&x)[8], const __half* w, int s, float eps) {
  float t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    t[i] = __fadd_rn(__fmul_rn(x[i], x[i]), __fmul_rn(x[4 + i], x[4 + i]));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = __fadd_rn(t[i], __shfl_xor_sync(0xffffffffu, t[i], o));
  const float ss = __fadd_rn(__fadd_rn(t[0], t[2]), __fadd_rn(t[1], t[3]));
  const float inv = 1.0f / sqrtf(__fadd_rn(__fdiv_rn(ss, 64.0f), eps));
  float wv[8];
  load4(w + 4 * s, wv);
  load4(w + 32 + 4 * s, wv + 4);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    x[i] = round_st<__half>(__fmul_rn(__fmul_rn(x[i], inv), wv[i]));
}

__device__ __forceinline__ void rotate_unit(float (&x)[8], const __half* rope, int s) {
  float cs[4], sn[4];
  load4(rope + 4 * s, cs);
  load4(rope + 32 + 4 * s, sn);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = x[i], b = x[4 + i];
    x[i] = round_st<__half>(__fsub_rn(__fmul_rn(a, cs[i]), __fmul_rn(b, sn[i])));
    x[4 + i] = round_st<__half>(__fadd_rn(__fmul_rn(b, cs[i]), __fmul_rn(a, sn[i])));
  }
}

__device__ __forceinline__ uint32_t pack_q8(const float* x, const float* sc, int per_channel) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float q = rintf(__fdiv_rn(x[i], per_channel ? sc[i] : sc[0]));
    w |= (uint32_t(int32_t(fminf(fmaxf(q, -128.f), 127.f))) & 0xffu) << (8 * i);
  }
  return w;
}

// One warp per (row, four consecutive units of its Hq + 2 Hkv).
template <int KVF>
__global__ void __launch_bounds__(kThreads)
    kv_append_kernel(const __grid_constant__ AppendArgs a) {
  const int lane = threadIdx.x & 31, s = lane & 7;
  const int units = a.hq + 2 * a.kv.hkv, groups = (units + 3) / 4;
  const int64_t item = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t row = item / groups;
  if (row >= a.at.n_rows) return;
  const int u = int(item - row * groups) * 4 + (lane >> 3);
  const bool is_q = u < a.hq, is_k = !is_q && u < a.hq + a.kv.hkv;
  const bool any = u < units && !(is_q && a.q_out == nullptr);
  float x[8] = {};
  if (any) {
    const __half* src = a.qkv + row * a.ld_qkv + u * 64;
    load4(src + 4 * s, x);
    load4(src + 32 + 4 * s, x + 4);
  }
  const int seq = warp_find_seq(a.at.row_start, a.at.nseq, row);
  if (seq < 0) return;  // behind the last sequence
  const SeqSpan span = seq_span(a.kv, a.at, seq);
  const int pos = span.past + int(row - span.row0);
  const int64_t at = span.ok ? kv_row(a.kv, seq, pos) : -1;
  if (at < 0) {
    if (lane == 0) atomicOr(a.err, kErrPosBeyondCache);
    return;
  }
  // the shuffles of the norm are warp-wide instructions: v units run them too and keep x
  if (a.norm_w != nullptr) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i];
    norm_unit(y, a.norm_w + (is_q ? 0 : 64), s, a.eps);
    if (is_q || is_k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = y[i];
    }
  }
  if (is_q || is_k) rotate_unit(x, a.rope + int64_t(pos) * 64, s);
  if (is_q && any) {
    __half* dst = a.q_out + row * a.ld_q + u * 64;
    store4(dst + 4 * s, x);
    store4(dst + 32 + 4 * s, x + 4);
  }
  const bool is_kv = !is_q && u < units;
  const int kh = u - a.hq - (is_k ? 0 : a.kv.hkv);
  unsigned char* base = (is_k ? a.kv.k : a.kv.v) + at * a.kv.row_bytes;
  if constexpr (KVF == kKvQ4) {
    q4_store_unit(x, reinterpret_cast<uint32_t*>(base + (is_kv ? kh : 0) * kQ4UnitBytes), is_kv);
  } else if (is_kv) {
    if constexpr (KVF == kKvF16) {
      __half* dst = reinterpret_cast<__half*>(base) + kh * 64;
      store4(dst + 4 * s, x);
      store4(dst + 32 + 4 * s, x + 4);
    } else {
      const float* sc = is_k ? a.kv.k_scale : a.kv.v_scale;
      if (a.kv.per_channel) sc += kh * 64 + 4 * s;
      const int far = a.kv.per_channel ? 32 : 0;
      uint32_t* dst = reinterpret_cast<uint32_t*>(base + kh * 64);
      dst[s] = pack_q8(x, sc, a.kv.per_channel);
      dst[8 + s] = pack_q8(x + 4, sc + far, a.kv.per_channel);
    }
  }
}

// One warp per (row, four consecutive units of K or V); lane s of a unit: dims 8s .. 8s+7.
template <int KVF>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadArgs a) {
  const int lane = threadIdx.x & 31, s = lane & 7;
  const int hkv = a.kv.hkv, units = 2 * hkv, groups = (units + 3) / 4;
  const int64_t item = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t row = item / groups;
  if (row >= a.at.n_rows) return;
  const int u = int(item - row * groups) * 4 + (lane >> 3);
  const int seq = warp_find_seq(a.at.row_start, a.at.nseq, row);
  if (seq < 0) return;
  const SeqSpan span = seq_span(a.kv, a.at, seq);
  const int64_t at = span.ok ? kv_row(a.kv, seq, span.past + int(row - span.row0)) : -1;
  if (at < 0) {
    if (lane == 0) atomicOr(a.err, kErrPosBeyondCache);
    return;
  }
  const bool is_k = u < hkv;
  const int kh = is_k ? u : u - hkv;
  __half* out = is_k ? a.k_out : a.v_out;
  if (u >= units || out == nullptr) return;
  const unsigned char* base = (is_k ? a.kv.k : a.kv.v) + at * a.kv.row_bytes;
  __half* dst = out + (row * hkv + kh) * 64 + 8 * s;
  if constexpr (KVF == kKvF16) {
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(base + kh * 128 + 16 * s);
  } else if constexpr (KVF == kKvI8) {
    const uint2 w = *reinterpret_cast<const uint2*>(base + kh * 64 + 8 * s);
    const float* sc = is_k ? a.kv.k_scale : a.kv.v_scale;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int8_t q = static_cast<int8_t>(((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 0xffu);
      v[i] = __fmul_rn(float(q), a.kv.per_channel ? sc[kh * 64 + 8 * s + i] : sc[0]);
    }
    store8(dst, v);
  } else {
    const uint32_t* unit = reinterpret_cast<const uint32_t*>(base + kh * kQ4UnitBytes);
    float sc, lo, v[8];
    q4_unpack(unit[8], sc, lo);
    q4_values(unit[s], sc, lo, v);
    store8(dst, v);
  }
}

// One warp per four consecutive (row, head) units of the dense source; the first unit's lanes of
// a row also clear the row's padding.
__global__ void __launch_bounds__(kThreads)
    quantize_q4_kernel(const __half* src, unsigned char* dst, int64_t units, int hkv,
                       int64_t row_bytes) {
  const int lane = threadIdx.x & 31, s = lane & 7;
  const int64_t warps = (int64_t(gridDim.x) * kThreads) >> 5;
  for (int64_t it = (int64_t(blockIdx.x) * kThreads + threadIdx.x) >> 5; it * 4 < units;
       it += warps) {
    const int64_t u = it * 4 + (lane >> 3);
    const bool any = u < units;
    const int64_t row = any ? u / hkv : 0;
    const int kh = int(u - row * hkv);
    float x[8] = {};
    if (any) {
      load4(src + u * 64 + 4 * s, x);
      load4(src + u * 64 + 32 + 4 * s, x + 4);
    }
    uint32_t* out = reinterpret_cast<uint32_t*>(dst + row * row_bytes);
    q4_store_unit(x, out + (any ? kh * 9 : 0), any);
    const int pad = int(row_bytes / 4) - hkv * 9;  // 0 .. 3 words
    if (any && kh == 0 && s < pad) out[hkv * 9 + s] = 0u;
  }
}

}  // namespace

cudaError_t launch_kv_append(const AppendArgs& a, cudaStream_t s) {
  const int64_t groups = (a.hq + 2 * a.kv.hkv + 3) / 4;
  const int64_t blocks = (a.at.n_rows * groups * 32 + kThreads - 1) / kThreads;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  const dim3 g{unsigned(blocks)};
  if (a.kv.format == kKvF16) kv_append_kernel<kKvF16><<<g, kThreads, 0, s>>>(a);
  else if (a.kv.format == kKvI8) kv_append_kernel<kKvI8><<<g, kThreads, 0, s>>>(a);
  else kv_append_kernel<kKvQ4><<<g, kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_kv_read(const ReadArgs& a, cudaStream_t s) {
  const int64_t groups = (2 * a.kv.hkv + 3) / 4;
  const int64_t blocks = (a.at.n_rows * groups * 32 + kThreads - 1) / kThreads;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  const dim3 g{unsigned(blocks)};
  if (a.kv.format == kKvF16) kv_read_kernel<kKvF16><<<g, kThreads, 0, s>>>(a);
  else if (a.kv.format == kKvI8) kv_read_kernel<kKvI8><<<g, kThreads, 0, s>>>(a);
  else kv_read_kernel<kKvQ4><<<g, kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_quantize_q4(const void* src, void* dst, int64_t rows, int hkv,
                               cudaStream_t s) {
  const int64_t units = rows * hkv;
  const int64_t want = (units * 8 + kThreads - 1) / kThreads;
  const int blocks = int(want < 148 * 16 ? want : 148 * 16);
  quantize_q4_kernel<<<blocks, kThreads, 0, s>>>(static_cast<const __half*>(src),
                                                 static_cast<unsigned char*>(dst), units, hkv,
                                                 q4_row_bytes(hkv));
  return cudaGetLastError();
}

}  // namespace p2p
