// logits_pick.cu -- penalties, biases and a grammar mask on a batch of logits and the greedy token
// of each row (the batched counterpart of ARGMAX, src/scripts/lfm-engine/kernels.js:362-399).
//
// A row's vocabulary is cut into the slices of one thread-block cluster; a CTA keeps the counts of
// its slice's tokens in shared memory and reads and writes its logits once, in 16-byte pieces whose
// first ones are loaded before the history is counted.
//   Histories of up to kLocalHist tokens are read whole by every CTA of the cluster, which counts
// the tokens of its slice: at most 16 KB out of L2 per CTA, against two cluster barriers.  Longer
// ones are read once per row: each CTA takes a part and counts every token straight into the owning
// CTA's shared memory (distributed shared memory).  Counts are whole numbers, so the order of the
// atomics does not matter.
//   Biased tokens are few: the streaming pass leaves them out, and a thread per token then does
// the whole computation with the token's biases in the order of the list.
// The CTAs' best tokens meet in the first CTA's shared memory, one slot each (a 64-bit maximum on
// distributed shared memory from several CTAs at once lost values).
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"

namespace p2p {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kMaxCluster = 8;
constexpr int kLocalHist = 4096;
constexpr int kMaxBiases = 512;            // of a slice, for the pass of their own
constexpr uint32_t kSeen = 0x80000000u;    // in the prompt (or generated: the count says so)
constexpr uint32_t kBiased = 0x40000000u;  // some bias entry names the token
constexpr uint32_t kCount = 0x3fffffffu;   // times generated
constexpr int kAhead = 4;                  // pieces of logits loaded before the history is read

// Larger value first, then smaller index; 0 is no token.  -0 and +0 are the same value.
__device__ __forceinline__ unsigned long long pick_key(float y, uint32_t v) {
  if (!(y > -INFINITY)) return 0ull;
  uint32_t b = __float_as_uint(y + 0.0f);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<unsigned long long>(b) << 32) | (0xffffffffu - v);
}

template <class T>
struct Piece {  // 16 bytes of logits
  static constexpr int kN = 16 / sizeof(T);
  uint4 w;
  __device__ __forceinline__ float get(int i) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    if constexpr (sizeof(T) == 4) return __uint_as_float(u[i]);
    const __half2 h = *reinterpret_cast<const __half2*>(&u[i >> 1]);
    return (i & 1) ? __high2float(h) : __low2float(h);
  }
  __device__ __forceinline__ void set(const float (&y)[kN]) {
    if constexpr (sizeof(T) == 4) {
      w = make_uint4(__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]),
                     __float_as_uint(y[3]));
    } else {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(y[2 * i], y[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
      w = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
};

struct Penalty {
  float rep, pres, freq;
  bool has_rep;
  __device__ __forceinline__ float apply(float x, uint32_t c) const {
    if (has_rep) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    if (c & kCount) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, float(c & kCount))), pres);
    return x;
  }
};

// Words in front of the counts of CTA `rank` of row i (its `pad`, see the kernel): slices are whole
// pieces apart, so all CTAs of a row have the same unless theirs ends before the boundary.
template <class T>
__device__ __forceinline__ int pad_of(const LogitsArgs& a, int i, int rank, int slice) {
  constexpr int kN = Piece<T>::kN;
  const uintptr_t p =
      reinterpret_cast<uintptr_t>(static_cast<const T*>(a.logits) + int64_t(i) * a.ld);
  const int n = min(slice, a.vocab - rank * slice);
  const int lead = min(n, int((16u - uint32_t(p & 15u)) & 15u) / int(sizeof(T)));
  return (kN - lead) % kN;
}

// cnt[] holds the slice's counts behind `pad` words, so that the counts of a 16-byte piece of
// logits start on 16 bytes whatever the row's alignment.
template <class T>
__global__ void __launch_bounds__(kThreads)
    logits_pick_kernel(const __grid_constant__ LogitsArgs a, int slice) {
  constexpr int kN = Piece<T>::kN;
  extern __shared__ __align__(16) uint32_t cnt[];  // [slice + kN]
  __shared__ unsigned long long warp_best[kThreads / 32];
  __shared__ unsigned long long cta_best[kMaxCluster];  // rank 0's: one slot per CTA
  __shared__ int bias_tok[kMaxBiases];
  __shared__ float bias_val[kMaxBiases], bias_x[kMaxBiases];
  __shared__ int warp_n[kThreads / 32];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = int(cl.block_rank()), csize = int(cl.num_blocks());
  const int i = blockIdx.x / csize, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int v0 = rank * slice, n = max(0, min(slice, a.vocab - v0));
  const T* src = static_cast<const T*>(a.logits) + int64_t(i) * a.ld + v0;
  T* dst = a.out ? static_cast<T*>(a.out) + int64_t(i) * a.ld_out + v0 : nullptr;
  // tokens in front of the first 16-byte boundary; whole pieces behind it
  const int lead =
      min(n, int((16u - uint32_t(reinterpret_cast<uintptr_t>(src) & 15u)) & 15u) / int(sizeof(T)));
  const int pad = (kN - lead) % kN, pieces = (n - lead) / kN;
  const uint4* body = reinterpret_cast<const uint4*>(src + lead);
  Piece<T> ahead[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (t + k * kThreads < pieces) ahead[k].w = body[t + k * kThreads];

  const bool remote = a.hist != nullptr && a.hist_cap > kLocalHist;
  for (int k = t; k < (slice + kN) / 4; k += kThreads)
    reinterpret_cast<uint4*>(cnt)[k] = make_uint4(0, 0, 0, 0);
  int len = 0, prompt = 0, e0 = 0, e1 = 0;
  if (a.hist != nullptr) {
    len = min(max(a.hist_len[i], 0), a.hist_cap);
    prompt = a.prompt_len ? a.prompt_len[i] : 0;
  }
  if (a.bias_start != nullptr) {
    e0 = min(max(a.bias_start[i], 0), a.n_bias);
    e1 = min(max(a.bias_start[i + 1], e0), a.n_bias);
  }
  Penalty pen;
  pen.has_rep = a.repetition != nullptr;
  pen.rep = a.repetition ? a.repetition[i] : 1.f;
  pen.pres = a.presence ? a.presence[i] : 0.f;
  pen.freq = a.frequency ? a.frequency[i] : 0.f;
  const int32_t* hist = a.hist + int64_t(i) * a.ld_hist;
  if (remote) cl.sync();
  else __syncthreads();
  if (remote) {
    for (int k = rank * kThreads + t; k < len; k += csize * kThreads) {
      const int v = hist[k];
      if (v < 0 || v >= a.vocab) continue;
      uint32_t* c = cl.map_shared_rank(cnt, v / slice) + pad_of<T>(a, i, v / slice, slice) +
                    v % slice;
      if (k >= prompt) atomicAdd(c, 1u);
      else atomicOr(c, kSeen);
    }
  } else {
#pragma unroll 4
    for (int k = t; k < len; k += kThreads) {
      const int v = hist[k] - v0;
      if (v < 0 || v >= n) continue;
      if (k >= prompt) atomicAdd(&cnt[pad + v], 1u);
      else atomicOr(&cnt[pad + v], kSeen);
    }
  }
  // the slice's biases, in the order of the list
  int n_bias = 0;
  bool scan = false;  // too many of them: the streaming pass looks each biased token up
  for (int k0 = e0; k0 < e1; k0 += kThreads) {
    const int k = k0 + t;
    const int v = k < e1 ? a.bias_tok[k] - v0 : -1;
    const bool mine = v >= 0 && v < n;
    const uint32_t votes = __ballot_sync(0xffffffffu, mine);
    if (lane == 0) warp_n[warp] = __popc(votes);
    __syncthreads();
    int at = n_bias + __popc(votes & ((1u << lane) - 1u));
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) at += warp_n[w];
      n_bias += warp_n[w];
    }
    if (mine && at < kMaxBiases) {
      bias_tok[at] = v;
      bias_val[at] = a.bias_val[k];
      bias_x[at] = to_f32(src[v]);  // before the streaming pass may store over it
    }
    __syncthreads();
  }
  scan = n_bias > kMaxBiases;
  if (remote) cl.sync();
  else __syncthreads();
  if (n_bias > 0) {  // the counts are complete
    if (scan) {
      for (int k = e0 + t; k < e1; k += kThreads) {
        const int v = a.bias_tok[k] - v0;
        if (v >= 0 && v < n) atomicOr(&cnt[pad + v], kBiased);
      }
    } else {
      for (int k = t; k < n_bias; k += kThreads) atomicOr(&cnt[pad + bias_tok[k]], kBiased);
    }
    __syncthreads();
  }
  const uint32_t* mask = a.mask ? a.mask + int64_t(i) * a.ld_mask : nullptr;
  unsigned long long best = 0ull;
  // the stored value of token v of the slice; biased ones are done later unless `scan`
  auto process = [&](float x, uint32_t c, int v, bool allowed) {
    if (c) {
      if (c & ~kBiased) x = pen.apply(x, c);
      if (scan && (c & kBiased)) {
        for (int k = e0; k < e1; ++k)
          if (a.bias_tok[k] == v0 + v) x = __fadd_rn(x, a.bias_val[k]);
      }
    }
    return to_f32(from_f32<T>(allowed ? x : -INFINITY));
  };
  auto consider = [&](float y, uint32_t c, int v) {
    if ((c & kBiased) && !scan) return;
    const unsigned long long key = pick_key(y, uint32_t(v0 + v));
    if (key > best) best = key;
  };
  auto allowed_bits = [&](int v) {  // of tokens v .. of the slice, at least kN of them
    if (mask == nullptr) return 0xffffffffu;
    const int g = v0 + v, w = g >> 5, sh = g & 31;
    uint32_t bits = mask[w] >> sh;
    if (sh + kN > 32 && (w + 1) * 32 < a.vocab) bits |= mask[w + 1] << (32 - sh);
    return bits;
  };
  const bool wide_out = dst != nullptr && (reinterpret_cast<uintptr_t>(dst + lead) & 15u) == 0;
  auto piece = [&](const Piece<T>& in, int k) {
    const int v = lead + k * kN;
    uint32_t c[kN];
#pragma unroll
    for (int j = 0; j < kN; j += 4) {
      const uint4 q = *reinterpret_cast<const uint4*>(&cnt[pad + v + j]);
      c[j] = q.x, c[j + 1] = q.y, c[j + 2] = q.z, c[j + 3] = q.w;
    }
    const uint32_t bits = allowed_bits(v);
    float y[kN], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      y[j] = process(in.get(j), c[j], v + j, (bits >> j) & 1u);
      if (!(c[j] & kBiased) || scan) top = fmaxf(top, y[j]);
    }
    // a piece whose best does not beat the thread's changes nothing (NaN never wins; an equal value
    // of a later token neither)
    if (pick_key(top, 0u) > best) {
#pragma unroll
      for (int j = 0; j < kN; ++j) consider(y[j], c[j], v + j);
    }
    if (dst != nullptr) {
      if (wide_out) {
        Piece<T> o;
        o.set(y);
        *reinterpret_cast<uint4*>(dst + v) = o.w;
      } else {
#pragma unroll
        for (int j = 0; j < kN; ++j) dst[v + j] = from_f32<T>(y[j]);
      }
    }
  };
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (t + k * kThreads < pieces) piece(ahead[k], t + k * kThreads);
  for (int k0 = t + kAhead * kThreads; k0 < pieces; k0 += kAhead * kThreads) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (k0 + k * kThreads < pieces) ahead[k].w = body[k0 + k * kThreads];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (k0 + k * kThreads < pieces) piece(ahead[k], k0 + k * kThreads);
  }
  // the tokens in front of and behind the pieces
  const int tail = lead + pieces * kN;
  for (int k = t; k < lead + (n - tail); k += kThreads) {
    const int v = k < lead ? k : tail + k - lead;
    const uint32_t c = cnt[pad + v];
    const float y = process(to_f32(src[v]), c, v, allowed_bits(v) & 1u);
    if (dst) dst[v] = from_f32<T>(y);
    consider(y, c, v);
  }
  if (n_bias > 0 && !scan) {
    __syncthreads();  // the pieces around them are stored
    for (int k = t; k < n_bias; k += kThreads) {
      const int v = bias_tok[k];
      bool first = true;
      for (int j = 0; j < k; ++j) first = first && bias_tok[j] != v;
      if (!first) continue;
      const uint32_t c = cnt[pad + v];
      float x = bias_x[k];
      if (c & ~kBiased) x = pen.apply(x, c);
      for (int j = k; j < n_bias; ++j)
        if (bias_tok[j] == v) x = __fadd_rn(x, bias_val[j]);
      if (!(allowed_bits(v) & 1u)) x = -INFINITY;
      const T y = from_f32<T>(x);
      if (dst) dst[v] = y;
      const unsigned long long key = pick_key(to_f32(y), uint32_t(v0 + v));
      if (key > best) best = key;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
    if (other > best) best = other;
  }
  if (lane == 0) warp_best[warp] = best;
  __syncthreads();
  if (t == 0) {
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w)
      if (warp_best[w] > best) best = warp_best[w];
    *cl.map_shared_rank(&cta_best[rank], 0) = best;
  }
  cl.sync();
  if (rank == 0 && t == 0) {
    unsigned long long k = 0ull;
    for (int r = 0; r < csize; ++r)
      if (cta_best[r] > k) k = cta_best[r];
    const int tok = k ? int(0xffffffffu - uint32_t(k & 0xffffffffull)) : -1;
    a.tok[i] = tok;
    if (a.advance && tok >= 0) {
      if (a.hist != nullptr && (a.hist_len[i] < 0 || a.hist_len[i] >= a.hist_cap)) {
        atomicOr(a.err, kErrHistFull);
      } else {
        if (a.hist != nullptr) {
          a.hist[int64_t(i) * a.ld_hist + len] = tok;
          a.hist_len[i] = len + 1;
        }
        if (a.past != nullptr) a.past[i] += 1;
      }
    }
  }
}

}  // namespace

cudaError_t launch_logits_pick(const LogitsArgs& a, int dtype, cudaStream_t s) {
  // slices of at least 1024 tokens, a multiple of 32 (whole mask words)
  int c = 1;
  while (c < kMaxCluster && a.vocab > c * 1024) c *= 2;
  const int slice = ((a.vocab + c - 1) / c + 31) / 32 * 32;
  const size_t smem = size_t(slice + 8) * 4;
  const void* fn = dtype == 0 ? reinterpret_cast<const void*>(&logits_pick_kernel<__half>)
                              : reinterpret_cast<const void*>(&logits_pick_kernel<float>);
  static PerDeviceOnce attrs[2];
  const cudaError_t e = per_device_once(attrs[dtype == 0 ? 0 : 1], [&](int&) {
    return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (((kMaxVocab + kMaxCluster - 1) / kMaxCluster + 31) / 32 * 32 + 8) * 4);
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(a.rows) * unsigned(c));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = unsigned(c);
  at.val.clusterDim.y = 1;
  at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  LogitsArgs arg = a;
  int sl = slice;
  void* args[] = {&arg, &sl};
  return cudaLaunchKernelExC(&cfg, fn, args);
}

}  // namespace p2p
