// logits_pick.cu -- penalties, biases and a grammar mask on a batch of logits and the greedy token
// of each row (the batched counterpart of ARGMAX, src/scripts/lfm-engine/kernels.js:362-399).
//
// A row's vocabulary is cut into the slices of one thread-block cluster.  The history is read once
// per row: each CTA takes a part of it and counts every token straight into the owning CTA's
// shared memory (distributed shared memory atomics), so a slice's counts are complete after one
// cluster barrier and the logits are then read and written once.  Counts are whole numbers and the
// maximum is order-free, so results do not depend on the order of the atomics.
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"

namespace p2p {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kMaxCluster = 8;
constexpr uint32_t kSeen = 0x80000000u;    // in the prompt (or generated: the count says so)
constexpr uint32_t kBiased = 0x40000000u;  // some bias entry names the token
constexpr uint32_t kCount = 0x3fffffffu;   // times generated

// Larger value first, then smaller index; 0 is no token.  -0 and +0 are the same value.
__device__ __forceinline__ unsigned long long pick_key(float y, uint32_t v) {
  if (!(y > -INFINITY)) return 0ull;
  uint32_t b = __float_as_uint(y + 0.0f);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<unsigned long long>(b) << 32) | (0xffffffffu - v);
}

template <class T>
__global__ void __launch_bounds__(kThreads)
    logits_pick_kernel(const __grid_constant__ LogitsArgs a, int slice, int vec) {
  extern __shared__ __align__(16) uint32_t cnt[];  // [slice]
  __shared__ unsigned long long warp_best[kThreads / 32];
  __shared__ unsigned long long cta_best[kMaxCluster];  // rank 0's: one slot per CTA
  cg::cluster_group cl = cg::this_cluster();
  const int rank = int(cl.block_rank()), csize = int(cl.num_blocks());
  const int i = blockIdx.x / csize, t = threadIdx.x;
  const int v0 = rank * slice, n = max(0, min(slice, a.vocab - v0));

  for (int k = t; k < slice / 4; k += kThreads)
    reinterpret_cast<uint4*>(cnt)[k] = make_uint4(0, 0, 0, 0);
  cl.sync();

  int len = 0, e0 = 0, e1 = 0;
  if (a.hist != nullptr) {
    len = min(max(a.hist_len[i], 0), a.hist_cap);
    const int prompt = a.prompt_len ? a.prompt_len[i] : 0;
    const int32_t* h = a.hist + int64_t(i) * a.ld_hist;
    for (int k = rank * kThreads + t; k < len; k += csize * kThreads) {
      const int v = h[k];
      if (v < 0 || v >= a.vocab) continue;
      uint32_t* c = cl.map_shared_rank(cnt, v / slice) + v % slice;
      if (k >= prompt) atomicAdd(c, 1u);
      else atomicOr(c, kSeen);
    }
  }
  if (a.bias_start != nullptr) {
    e0 = min(max(a.bias_start[i], 0), a.n_bias);
    e1 = min(max(a.bias_start[i + 1], e0), a.n_bias);
  }
  cl.sync();
  if (e1 > e0) {  // the counts are complete: marks of this slice's biased tokens
    for (int k = e0 + t; k < e1; k += kThreads) {
      const int v = a.bias_tok[k] - v0;
      if (v >= 0 && v < n) atomicOr(&cnt[v], kBiased);
    }
    __syncthreads();
  }
  const float rep = a.repetition ? a.repetition[i] : 1.f;
  const float pres = a.presence ? a.presence[i] : 0.f;
  const float freq = a.frequency ? a.frequency[i] : 0.f;
  const T* src = static_cast<const T*>(a.logits) + int64_t(i) * a.ld + v0;
  T* dst = a.out ? static_cast<T*>(a.out) + int64_t(i) * a.ld_out + v0 : nullptr;
  const uint32_t* mask = a.mask ? a.mask + int64_t(i) * a.ld_mask + v0 / 32 : nullptr;
  unsigned long long best = 0ull;
  for (int v = t; v < n; v += kThreads) {
    float x = to_f32(src[v]);
    const uint32_t c = cnt[v];
    if (c & ~kBiased) {
      if (a.repetition) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      if (c & kCount) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, float(c & kCount))), pres);
    }
    if (c & kBiased) {
      for (int k = e0; k < e1; ++k)
        if (a.bias_tok[k] == v0 + v) x = __fadd_rn(x, a.bias_val[k]);
    }
    if (mask && !((mask[v >> 5] >> (v & 31)) & 1u)) x = -INFINITY;
    const T y = from_f32<T>(x);
    if (dst) dst[v] = y;
    const unsigned long long key = pick_key(to_f32(y), uint32_t(v0 + v));
    if (key > best) best = key;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
    if (other > best) best = other;
  }
  if ((t & 31) == 0) warp_best[t >> 5] = best;
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
  const size_t smem = size_t(slice) * 4;
  const void* fn = dtype == 0 ? reinterpret_cast<const void*>(&logits_pick_kernel<__half>)
                              : reinterpret_cast<const void*>(&logits_pick_kernel<float>);
  static PerDeviceOnce attrs[2];
  const cudaError_t e = per_device_once(attrs[dtype == 0 ? 0 : 1], [&](int&) {
    return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                ((kMaxVocab + kMaxCluster - 1) / kMaxCluster + 31) / 32 * 32 * 4);
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
  int sl = slice, vec = 0;
  void* args[] = {&arg, &sl, &vec};
  return cudaLaunchKernelExC(&cfg, fn, args);
}

}  // namespace p2p
