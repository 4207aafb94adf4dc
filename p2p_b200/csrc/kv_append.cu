// kv_append.cu -- rows of ragged prompt chunks into a KV cache of any layout (QK_PREP,
// src/scripts/lfm-engine/kernels.js:216-266, with the append generalised), cached sequences read
// back, and f16 rows to the 4-bit format.
//
// All three move bytes and compute little.  A unit -- the 64 values of one (row, head) -- belongs
// to 8 lanes, so a warp works on four units at a time and each of its loads and stores covers whole
// 32-byte sectors: lane s of a unit holds dims 4s .. 4s+3 and 32+4s .. 32+4s+3, which are
// rotate-half partners, so the rotation needs no exchange.  A warp has up to kIter such groups of
// one row: their loads are all on their way before the row's sequence, position, page and rope row
// are looked up, one after the other, once for all of them.
//   Bound by issue: 12 prompts (11.4k rows of 32 + 8 + 8 heads, 142 MB) take 35 us, 62 % of the copy rate,
// at 83 % of the issue slots (225 instructions a group); small calls by latency (one row: 2.8 us).  4-bit
// units halve the bytes written but not the instructions (509 rows appended and read back: 10.1 us).
#include "common.cuh"
#include "kernels.h"
#include "kv_view.cuh"

namespace p2p {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void widen4(const uint2& w, float* v) {
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
  v[0] = a.x;
  v[1] = a.y;
  v[2] = b.x;
  v[3] = b.y;
}
__device__ __forceinline__ void load4(const __half* p, float* v) {
  widen4(*reinterpret_cast<const uint2*>(p), v);
}
__device__ __forceinline__ uint2 round4(float a, float b, float c, float d) {
  const __half2 x = __floats2half2_rn(a, b), y = __floats2half2_rn(c, d);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

// The sum of squares of a unit (x: 8 values per lane), in the shader's tree (kernels.js:246-251:
// t[i] = v[i]^2 + v[i+32]^2, then pairs 16, 8, 4, 2, 1 apart), each IEEE operation on its own, so it is bit-identical to it (an addition's order of operands
// does not matter).  Lane l holds t[4l .. 4l+3]: pairs 16 and 8 apart lie 4 and 2 lanes away, and a
// lane keeps only half of its sums at each of these steps.
__device__ __forceinline__ float square_sum(const float (&x)[8], int s) {
  float t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    t[i] = __fadd_rn(__fmul_rn(x[i], x[i]), __fmul_rn(x[4 + i], x[4 + i]));
  const bool up = (s & 4) != 0, odd = (s & 2) != 0;
  // 16 apart: the lower lane keeps sums 0, 1, the upper one 2, 3
  const float g0 = __shfl_xor_sync(0xffffffffu, up ? t[0] : t[2], 4);
  const float g1 = __shfl_xor_sync(0xffffffffu, up ? t[1] : t[3], 4);
  const float p0 = __fadd_rn(up ? t[2] : t[0], g0), p1 = __fadd_rn(up ? t[3] : t[1], g1);
  // 8 apart: one of the two
  const float g2 = __shfl_xor_sync(0xffffffffu, odd ? p0 : p1, 2);
  float r = __fadd_rn(odd ? p1 : p0, g2);
  r = __fadd_rn(r, __shfl_xor_sync(0xffffffffu, r, 1));  // 4 apart
  r = __fadd_rn(r, __shfl_xor_sync(0xffffffffu, r, 4));  // 2 apart: sums c and c + 2
  return __fadd_rn(r, __shfl_xor_sync(0xffffffffu, r, 2));  // 1 apart
}

// x normed with the weights w (packed) and rounded to f16.
__device__ __forceinline__ void norm_unit(float (&x)[8], const uint2 (&w)[2], float inv) {
  float f[8];
  widen4(w[0], f);
  widen4(w[1], f + 4);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 y = __half22float2(__floats2half2_rn(
        __fmul_rn(__fmul_rn(x[i], inv), f[i]), __fmul_rn(__fmul_rn(x[i + 1], inv), f[i + 1])));
    x[i] = y.x;
    x[i + 1] = y.y;
  }
}

// The rotate-half RoPE of a unit's dims i and 32 + i, rounded to f16.
__device__ __forceinline__ void rotate_unit(const float (&x)[8], const float (&cs)[4],
                                            const float (&sn)[4], uint2& lo, uint2& hi) {
  float a[4], b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = __fsub_rn(__fmul_rn(x[i], cs[i]), __fmul_rn(x[4 + i], sn[i]));
    b[i] = __fadd_rn(__fmul_rn(x[4 + i], cs[i]), __fmul_rn(x[i], sn[i]));
  }
  lo = round4(a[0], a[1], a[2], a[3]);
  hi = round4(b[0], b[1], b[2], b[3]);
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

// The first block of a launch reports the sequences that do not fit, by themselves: those whose rows
// all lie behind n_rows, or that a falling row_start leaves without any, belong to no row's warp.
__device__ __forceinline__ void report_misfits(const KvView& kv, const ChunkIndex& at, int32_t* err) {
  bool bad = false;
  for (int z = threadIdx.x; z < at.nseq; z += kThreads) {
    const SeqSpan span = seq_span(kv, at, z);
    bad |= span.len != 0 && !span.ok;
  }
  if (bad) atomicOr(err, kErrPosBeyondCache);
}

// One warp per (row, 4 kIter consecutive units of its Hq + 2 Hkv).
template <int KVF, int kIter>
__global__ void __launch_bounds__(kThreads)
    kv_append_kernel(const __grid_constant__ AppendArgs a) {
  if (blockIdx.x == 0) return report_misfits(a.kv, a.at, a.err);
  const int lane = threadIdx.x & 31, s = lane & 7;
  const int units = a.hq + 2 * a.kv.hkv, groups = (units + 4 * kIter - 1) / (4 * kIter);
  const int64_t item = (int64_t(blockIdx.x - 1) * kThreads + threadIdx.x) >> 5;
  const int64_t row = item / groups;
  if (row >= a.at.n_rows) return;
  const int u0 = int(item - row * groups) * 4 * kIter + (lane >> 3);
  const __half* src = a.qkv + row * a.ld_qkv + 4 * s;
  uint2 raw[kIter][2];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int u = u0 + 4 * i;
    raw[i][0] = raw[i][1] = make_uint2(0u, 0u);
    if (u < units && !(u < a.hq && a.q_out == nullptr)) {
      raw[i][0] = *reinterpret_cast<const uint2*>(src + u * 64);
      raw[i][1] = *reinterpret_cast<const uint2*>(src + u * 64 + 32);
    }
  }
  const int seq = warp_find_seq(a.at.row_start, a.at.nseq, row);
  if (seq < 0) return;  // no sequence's row
  const SeqSpan span = seq_span(a.kv, a.at, seq);
  const int pos = span.past + int(row - span.row0);
  const int64_t at = span.ok ? kv_row(a.kv, seq, pos) : -1;
  if (at < 0) {
    if (lane == 0) atomicOr(a.err, kErrPosBeyondCache);
    return;
  }
  float cs[4], sn[4];
  load4(a.rope + int64_t(pos) * 64 + 4 * s, cs);
  load4(a.rope + int64_t(pos) * 64 + 32 + 4 * s, sn);
  const bool norm = a.norm_w != nullptr;
  uint2 wq[2] = {}, wk[2] = {};  // this lane's norm weights of q and of k units
  float inv = 0.f;
  if (norm) {
    const __half* nw = a.norm_w + 4 * s;
    wq[0] = *reinterpret_cast<const uint2*>(nw);
    wq[1] = *reinterpret_cast<const uint2*>(nw + 32);
    wk[0] = *reinterpret_cast<const uint2*>(nw + 64);
    wk[1] = *reinterpret_cast<const uint2*>(nw + 96);
    // lane s works out 1 / sqrt for group s % kIter; the others take it from there
    float mean = 0.f;
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      float x[8];
      widen4(raw[i][0], x);
      widen4(raw[i][1], x + 4);
      const float r = square_sum(x, s);
      if (s % kIter == i) mean = __fmul_rn(r, 0.015625f);
    }
    inv = __frcp_rn(__fsqrt_rn(__fadd_rn(mean, a.eps)));
  }
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int u = u0 + 4 * i, first = u - (lane >> 3);
    if (first >= units) break;  // the warp's units end before
    const bool is_q = u < a.hq, is_k = !is_q && u < a.hq + a.kv.hkv;
    uint2 lo = raw[i][0], hi = raw[i][1];
    if (first < a.hq + a.kv.hkv) {  // not v units alone
      float x[8];
      widen4(lo, x);
      widen4(hi, x + 4);
      if (norm) {
        const float mine = __shfl_sync(0xffffffffu, inv, (lane & 24) + i);
        const uint2 w[2] = {is_q ? wq[0] : wk[0], is_q ? wq[1] : wk[1]};
        norm_unit(x, w, mine);
      }
      if (is_q || is_k) rotate_unit(x, cs, sn, lo, hi);
    }
    if (is_q && a.q_out != nullptr) {
      __half* dst = a.q_out + row * a.ld_q + u * 64 + 4 * s;
      *reinterpret_cast<uint2*>(dst) = lo;
      *reinterpret_cast<uint2*>(dst + 32) = hi;
    }
    if (first + 3 < a.hq) continue;  // q units alone
    const bool is_kv = !is_q && u < units;
    const int kh = u - a.hq - (is_k ? 0 : a.kv.hkv);
    unsigned char* base = (is_k ? a.kv.k : a.kv.v) + at * a.kv.row_bytes;
    if constexpr (KVF == kKvF16) {
      if (is_kv) {
        __half* dst = reinterpret_cast<__half*>(base) + kh * 64 + 4 * s;
        *reinterpret_cast<uint2*>(dst) = lo;
        *reinterpret_cast<uint2*>(dst + 32) = hi;
      }
    } else {
      float x[8];
      widen4(lo, x);
      widen4(hi, x + 4);
      if constexpr (KVF == kKvQ4) {
        q4_store_unit(x, reinterpret_cast<uint32_t*>(base + (is_kv ? kh : 0) * kQ4UnitBytes),
                      is_kv);
      } else if (is_kv) {
        const float* sc = is_k ? a.kv.k_scale : a.kv.v_scale;
        if (a.kv.per_channel) sc += kh * 64 + 4 * s;
        const int far = a.kv.per_channel ? 32 : 0;
        uint32_t* dst = reinterpret_cast<uint32_t*>(base + kh * 64);
        dst[s] = pack_q8(x, sc, a.kv.per_channel);
        dst[8 + s] = pack_q8(x + 4, sc + far, a.kv.per_channel);
      }
    }
  }
}

// One warp per (row, 4 kIter consecutive units of K and V); lane s of a unit: dims 8s .. 8s+7.
template <int KVF, int kIter>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadArgs a) {
  if (blockIdx.x == 0) return report_misfits(a.kv, a.at, a.err);
  const int lane = threadIdx.x & 31, s = lane & 7;
  const int hkv = a.kv.hkv, units = 2 * hkv, groups = (units + 4 * kIter - 1) / (4 * kIter);
  const int64_t item = (int64_t(blockIdx.x - 1) * kThreads + threadIdx.x) >> 5;
  const int64_t row = item / groups;
  if (row >= a.at.n_rows) return;
  const int seq = warp_find_seq(a.at.row_start, a.at.nseq, row);
  if (seq < 0) return;
  const SeqSpan span = seq_span(a.kv, a.at, seq);
  const int64_t at = span.ok ? kv_row(a.kv, seq, span.past + int(row - span.row0)) : -1;
  if (at < 0) {
    if (lane == 0) atomicOr(a.err, kErrPosBeyondCache);
    return;
  }
  const int u0 = int(item - row * groups) * 4 * kIter + (lane >> 3);
  uint4 raw[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int u = u0 + 4 * i;
    if (u >= units || (u < hkv ? a.k_out : a.v_out) == nullptr) continue;
    const unsigned char* base = (u < hkv ? a.kv.k : a.kv.v) + at * a.kv.row_bytes;
    const int kh = u < hkv ? u : u - hkv;
    if constexpr (KVF == kKvF16) {
      raw[i] = *reinterpret_cast<const uint4*>(base + kh * 128 + 16 * s);
    } else if constexpr (KVF == kKvI8) {
      const uint2 w = *reinterpret_cast<const uint2*>(base + kh * 64 + 8 * s);
      raw[i].x = w.x;
      raw[i].y = w.y;
    } else {
      const uint32_t* unit = reinterpret_cast<const uint32_t*>(base + kh * kQ4UnitBytes);
      raw[i].x = unit[s];
      raw[i].y = unit[8];
    }
  }
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int u = u0 + 4 * i;
    __half* out = u < hkv ? a.k_out : a.v_out;
    if (u >= units || out == nullptr) continue;
    const int kh = u < hkv ? u : u - hkv;
    __half* dst = out + (row * hkv + kh) * 64 + 8 * s;
    if constexpr (KVF == kKvF16) {
      *reinterpret_cast<uint4*>(dst) = raw[i];
    } else if constexpr (KVF == kKvI8) {
      const float* sc = u < hkv ? a.kv.k_scale : a.kv.v_scale;
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int8_t q =
            static_cast<int8_t>(((k < 4 ? raw[i].x : raw[i].y) >> (8 * (k & 3))) & 0xffu);
        v[k] = __fmul_rn(float(q), a.kv.per_channel ? sc[kh * 64 + 8 * s + k] : sc[0]);
      }
      store8(dst, v);
    } else {
      float sc, lo, v[8];
      q4_unpack(raw[i].y, sc, lo);
      q4_values(raw[i].x, sc, lo, v);
      store8(dst, v);
    }
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

// A warp takes four groups of units of a row when that still fills the SMs' 32 warps twice over
// (11.4k rows of 48 units into f16 pages: 35 us against 46 with one), else one (1 row: 2.8 us against
// 3.7).
static bool wide(int64_t rows, int64_t units, int num_sms) {
  return rows * ((units + 15) / 16) >= int64_t(num_sms) * 32 * 2;
}
template <template <int, int> class K, class A>
static cudaError_t launch_rows(const A& a, int64_t units, int num_sms, cudaStream_t s) {
  const bool w = wide(a.at.n_rows, units, num_sms);
  const int64_t groups = w ? (units + 15) / 16 : (units + 3) / 4;
  const int64_t blocks = (a.at.n_rows * groups * 32 + kThreads - 1) / kThreads;
  if (blocks >= INT32_MAX) return cudaErrorInvalidValue;
  const dim3 g{unsigned(blocks + 1)};  // and the one that reports
  if (a.kv.format == kKvF16) w ? K<kKvF16, 4>::run(g, s, a) : K<kKvF16, 1>::run(g, s, a);
  else if (a.kv.format == kKvI8) w ? K<kKvI8, 4>::run(g, s, a) : K<kKvI8, 1>::run(g, s, a);
  else w ? K<kKvQ4, 4>::run(g, s, a) : K<kKvQ4, 1>::run(g, s, a);
  return cudaGetLastError();
}
template <int KVF, int IT>
struct Append {
  static void run(dim3 g, cudaStream_t s, const AppendArgs& a) {
    kv_append_kernel<KVF, IT><<<g, kThreads, 0, s>>>(a);
  }
};
template <int KVF, int IT>
struct Read {
  static void run(dim3 g, cudaStream_t s, const ReadArgs& a) {
    kv_read_kernel<KVF, IT><<<g, kThreads, 0, s>>>(a);
  }
};

cudaError_t launch_kv_append(const AppendArgs& a, int num_sms, cudaStream_t s) {
  return launch_rows<Append>(a, a.hq + 2 * a.kv.hkv, num_sms, s);
}

cudaError_t launch_kv_read(const ReadArgs& a, int num_sms, cudaStream_t s) {
  return launch_rows<Read>(a, 2 * a.kv.hkv, num_sms, s);
}

cudaError_t launch_quantize_q4(const void* src, void* dst, int64_t rows, int hkv, int num_sms,
                               cudaStream_t s) {
  const int64_t units = rows * hkv;
  const int64_t want = (units * 8 + kThreads - 1) / kThreads;
  const int blocks = int(want < num_sms * 16 ? want : num_sms * 16);
  quantize_q4_kernel<<<blocks, kThreads, 0, s>>>(static_cast<const __half*>(src),
                                                 static_cast<unsigned char*>(dst), units, hkv,
                                                 q4_row_bytes(hkv));
  return cudaGetLastError();
}

}  // namespace p2p
