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
//   The touched tokens -- penalised or biased -- are few.  Threads take one each, compute its value in
// f32 and leave it in the token's count word, with a bit in a map of the slice; the streaming pass
// looks at the map and otherwise only masks, stores and compares.  (With the penalties in the
// streaming pass nearly every warp ran their divisions for one lane or another: 74 instructions per
// token.)
//   One row of 65536 f16 logits takes 4.6 us, which is latency (launch, history, counts, stream, cluster
// barrier); 64 rows with everything 11.4 us; 128 rows of 131071 f32 logits, 4000 tokens of history and 300
// biases each, 59 us (2.3 TB/s): two CTAs per SM, which is what the counts leave room for, wait at their
// barriers.
// The CTAs' best tokens meet in the first CTA's shared memory, one slot each (a 64-bit maximum on
// distributed shared memory from several CTAs at once lost values).
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"

namespace p2p {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxCluster = 8;
constexpr int kLocalHist = 4096;
// Threads of a CTA: 256 up to this slice (four CTAs per SM: 64 rows of 65536 in 11.4 us, 15.8 with
// 512), 512 above, where the counts leave room for two CTAs (128 rows of 131071 f32 in 59 us, 73 with
// 256).
constexpr int kSmallSlice = 12288;
constexpr uint32_t kSeen = 0x80000000u;    // in the prompt (or generated: the count says so)
constexpr uint32_t kCount = 0x7fffffffu;   // times generated
constexpr int kAhead = 4;                  // pieces of logits loaded before the history is read

// Larger value first, then smaller index; 0 is no token (y = -inf).  -0 and +0 are the same value.
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

template <class T, int kThreads>
__global__ void __launch_bounds__(kThreads)
    logits_pick_kernel(const __grid_constant__ LogitsArgs a, int slice) {
  constexpr int kN = Piece<T>::kN;
  // per token of the slice a count, later the value of a touched token; a bit each: touched, allowed;
  // the counted tokens (short histories)
  extern __shared__ __align__(16) uint32_t cnt[];
  uint32_t* map = cnt + (a.hist != nullptr || a.bias_start != nullptr ? slice : 0);
  uint32_t* mask = map + slice / 32;
  uint16_t* list = reinterpret_cast<uint16_t*>(mask + slice / 32);
  __shared__ float warp_y[kThreads / 32];
  __shared__ uint32_t warp_v[kThreads / 32];
  __shared__ unsigned long long cta_best[kMaxCluster];  // rank 0's: one slot per CTA
  __shared__ int bias_tok[kThreads];
  __shared__ float bias_val[kThreads];
  __shared__ int warp_n[kThreads / 32];
  __shared__ int n_list;
  cg::cluster_group cl = cg::this_cluster();
  const int rank = int(cl.block_rank()), csize = int(cl.num_blocks());
  const int i = blockIdx.x / csize, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int v0 = rank * slice, n = max(0, min(slice, a.vocab - v0));
  const T* src = static_cast<const T*>(a.logits) + int64_t(i) * a.ld + v0;
  T* dst = a.out ? static_cast<T*>(a.out) + int64_t(i) * a.ld_out + v0 : nullptr;
  // tokens in front of the first 16-byte boundary; whole pieces behind it
  const int lead =
      min(n, int((16u - uint32_t(reinterpret_cast<uintptr_t>(src) & 15u)) & 15u) / int(sizeof(T)));
  const int pieces = (n - lead) / kN;
  const uint4* body = reinterpret_cast<const uint4*>(src + lead);
  Piece<T> ahead[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (t + k * kThreads < pieces) ahead[k].w = body[t + k * kThreads];

  // Another CTA's shared memory is not touched before that CTA runs: everyone reports here and waits
  // in front of the first access.
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  // ... and everything else the CTA is going to look at is asked for now, before any of it is
  // needed: the row's history (short ones whole; what lies behind its length is dropped later), the
  // first of its biases, the slice's mask words
  const bool remote = a.hist != nullptr && a.hist_cap > kLocalHist;
  const int32_t* hist = a.hist + int64_t(i) * a.ld_hist;
  constexpr int kHist = kLocalHist / kThreads;
  int early[kHist];
  if (a.hist != nullptr && !remote) {
#pragma unroll
    for (int k = 0; k < kHist; ++k)
      early[k] = t + k * kThreads < a.hist_cap ? hist[t + k * kThreads] : -1;
  }
  const int words = a.mask ? (n + 31) / 32 : 0;
  const uint32_t* mask_row = a.mask ? a.mask + int64_t(i) * a.ld_mask + v0 / 32 : nullptr;
  const uint32_t early_mask = t < words ? mask_row[t] : 0u;
  int len = 0, prompt = 0, e0 = 0, e1 = 0;
  if (a.hist != nullptr) {
    len = min(max(a.hist_len[i], 0), a.hist_cap);
    prompt = a.prompt_len ? a.prompt_len[i] : 0;
  }
  if (a.bias_start != nullptr) {
    e0 = min(max(a.bias_start[i], 0), a.n_bias);
    e1 = min(max(a.bias_start[i + 1], e0), a.n_bias);
  }
  const int early_tok = e0 + t < e1 ? a.bias_tok[e0 + t] : -1;
  const float early_val = e0 + t < e1 ? a.bias_val[e0 + t] : 0.f;
  if (t < words) mask[t] = early_mask;
  for (int k = t + kThreads; k < words; k += kThreads) mask[k] = mask_row[k];
  const bool touched = a.hist != nullptr || a.bias_start != nullptr;
  if (touched) {
    const bool has_rep = a.repetition != nullptr;
    const float rep = has_rep ? a.repetition[i] : 1.f;
    const float pres = a.presence ? a.presence[i] : 0.f;
    const float freq = a.frequency ? a.frequency[i] : 0.f;
    for (int k = t; k < (slice + slice / 32) / 4; k += kThreads)
      reinterpret_cast<uint4*>(cnt)[k] = make_uint4(0, 0, 0, 0);
    if (t == 0) n_list = 0;
    if (remote) {
      asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
      cl.sync();  // the counts are clear
    } else {
      __syncthreads();
    }
    if (remote) {
      for (int k = rank * kThreads + t; k < len; k += csize * kThreads) {
        const int v = hist[k];
        if (v < 0 || v >= a.vocab) continue;
        uint32_t* c = cl.map_shared_rank(cnt, v / slice) + v % slice;
        if (k >= prompt) atomicAdd(c, 1u);
        else atomicOr(c, kSeen);
      }
      cl.sync();
    } else {
#pragma unroll
      for (int j = 0; j < kHist; ++j) {
        if (j * kThreads >= len) break;
        const int k = t + j * kThreads, v = early[j] - v0;
        bool fresh = false;
        if (k < len && v >= 0 && v < n)
          fresh = (k >= prompt ? atomicAdd(&cnt[v], 1u) : atomicOr(&cnt[v], kSeen)) == 0u;
        // the first to touch a token lists it; one count a warp
        const uint32_t votes = __ballot_sync(0xffffffffu, fresh);
        int at = 0;
        if (lane == 0 && votes) at = atomicAdd(&n_list, __popc(votes));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(votes & ((1u << lane) - 1u));
        if (fresh) list[at] = uint16_t(v);
      }
      __syncthreads();
    }
    auto penalise = [&](int v, float x) {
      const uint32_t c = cnt[v];
      if (has_rep) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      if (c & kCount) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, float(c & kCount))), pres);
      cnt[v] = __float_as_uint(x);
      atomicOr(&map[v >> 5], 1u << (v & 31));
    };
    if (remote) {
      for (int v = t; v < n; v += kThreads)
        if (cnt[v] != 0u) penalise(v, to_f32(src[v]));
    } else {
      for (int k0 = t; k0 < n_list; k0 += 4 * kThreads) {  // four logits on their way
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (k0 + j * kThreads < n_list) x[j] = to_f32(src[list[k0 + j * kThreads]]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (k0 + j * kThreads < n_list) penalise(list[k0 + j * kThreads], x[j]);
      }
    }
    // the slice's biases, in the order of the list, a round of kThreads entries at a time
    for (int k0 = e0; k0 < e1; k0 += kThreads) {
      const int k = k0 + t;
      const int tok = k0 == e0 ? early_tok : k < e1 ? a.bias_tok[k] : -1;
      const int v = tok - v0;
      const bool mine = tok >= 0 && v >= 0 && v < n;
      const uint32_t votes = __ballot_sync(0xffffffffu, mine);
      if (lane == 0) warp_n[warp] = __popc(votes);
      __syncthreads();  // also: the penalties, or the round before, are in place
      int at = __popc(votes & ((1u << lane) - 1u)), all = 0;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) at += warp_n[w];
        all += warp_n[w];
      }
      if (mine) {
        bias_tok[at] = v;
        bias_val[at] = k0 == e0 ? early_val : a.bias_val[k];
      }
      __syncthreads();
      if (t < all) {  // a token's first entry adds all of them, in order
        const int u = bias_tok[t];
        bool first = true;
        for (int j = 0; j < t; ++j) first = first && bias_tok[j] != u;
        if (first) {
          const bool known = (map[u >> 5] >> (u & 31)) & 1u;
          float x = known ? __uint_as_float(cnt[u]) : to_f32(src[u]);
          for (int j = t; j < all; ++j)
            if (bias_tok[j] == u) x = __fadd_rn(x, bias_val[j]);
          cnt[u] = __float_as_uint(x);
          atomicOr(&map[u >> 5], 1u << (u & 31));
        }
      }
      __syncthreads();
    }
  }
  __syncthreads();
  // bits of the kN tokens from v on, out of a word a 32 tokens (v0 is a multiple of 32)
  auto bits_of = [&](const uint32_t* words, int v) {
    const int w = v >> 5, sh = v & 31;
    uint32_t bits = words[w] >> sh;
    if (sh + kN > 32 && (w + 1) * 32 < n) bits |= words[w + 1] << (32 - sh);
    return bits;
  };
  float best = -INFINITY;  // NaN and -inf never win
  uint32_t best_v = 0xffffffffu;
  const bool wide_out = dst != nullptr && (reinterpret_cast<uintptr_t>(dst + lead) & 15u) == 0;
  auto piece = [&](Piece<T> in, int k) {
    const int v = lead + k * kN;
    float y[kN];
#pragma unroll
    for (int j = 0; j < kN; ++j) y[j] = in.get(j);
    const uint32_t hit = touched ? bits_of(map, v) & ((1u << kN) - 1u) : 0u;
    if (hit) {
#pragma unroll
      for (int j = 0; j < kN; ++j)
        if ((hit >> j) & 1u) y[j] = round_st<T>(__uint_as_float(cnt[v + j]));
    }
    if (words) {
      const uint32_t bits = bits_of(mask, v);
#pragma unroll
      for (int j = 0; j < kN; ++j)
        if (!((bits >> j) & 1u)) y[j] = -INFINITY;
    }
    float top = y[0];
#pragma unroll
    for (int j = 1; j < kN; ++j) top = fmaxf(top, y[j]);
    if (top > best) {  // a thread's pieces come in the order of their tokens
      best = top;
#pragma unroll
      for (int j = kN - 1; j >= 0; --j)
        if (y[j] == top) best_v = uint32_t(v0 + v + j);
    }
    if (dst != nullptr) {
      if (wide_out) {
        in.set(y);
        *reinterpret_cast<uint4*>(dst + v) = in.w;
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
    float y = to_f32(src[v]);
    if (touched && ((map[v >> 5] >> (v & 31)) & 1u)) y = round_st<T>(__uint_as_float(cnt[v]));
    if (words && !((mask[v >> 5] >> (v & 31)) & 1u)) y = -INFINITY;
    if (dst) dst[v] = from_f32<T>(y);
    if (y > best || (y == best && uint32_t(v0 + v) < best_v)) {
      best = y;
      best_v = uint32_t(v0 + v);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float y = __shfl_xor_sync(0xffffffffu, best, o);
    const uint32_t v = __shfl_xor_sync(0xffffffffu, best_v, o);
    if (y > best || (y == best && v < best_v)) {
      best = y;
      best_v = v;
    }
  }
  if (lane == 0) {
    warp_y[warp] = best;
    warp_v[warp] = best_v;
  }
  if (!remote) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  __syncthreads();
  if (t == 0) {
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w)
      if (warp_y[w] > best || (warp_y[w] == best && warp_v[w] < best_v)) {
        best = warp_y[w];
        best_v = warp_v[w];
      }
    *cl.map_shared_rank(&cta_best[rank], 0) = pick_key(best, best_v);
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
  // slices of at least 1024 tokens, a multiple of 128 (whole words of masks and 16 bytes of the map)
  int c = 1;
  while (c < kMaxCluster && a.vocab > c * 1024) c *= 2;
  const int slice = ((a.vocab + c - 1) / c + 127) / 128 * 128;
  constexpr int kMaxSlice = ((kMaxVocab + kMaxCluster - 1) / kMaxCluster + 127) / 128 * 128;
  static_assert(kMaxSlice <= 65536, "a slice's tokens in 16 bits");
  auto bytes = [](int slice, int hist) {
    return size_t(slice) * 4 + size_t(slice) / 4 + size_t(hist) * 2;
  };
  const bool touched = a.hist != nullptr || a.bias_start != nullptr;
  const bool listed = a.hist != nullptr && a.hist_cap <= kLocalHist;
  const size_t smem = touched ? bytes(slice, listed ? a.hist_cap : 0) : size_t(slice) / 4;
  const int which = (dtype == 0 ? 0 : 2) + (slice > kSmallSlice ? 1 : 0);
  const int threads = slice > kSmallSlice ? 512 : 256;
  const void* fn = which == 0   ? reinterpret_cast<const void*>(&logits_pick_kernel<__half, 256>)
                   : which == 1 ? reinterpret_cast<const void*>(&logits_pick_kernel<__half, 512>)
                   : which == 2 ? reinterpret_cast<const void*>(&logits_pick_kernel<float, 256>)
                                : reinterpret_cast<const void*>(&logits_pick_kernel<float, 512>);
  static PerDeviceOnce attrs[4];
  const cudaError_t e = per_device_once(attrs[which], [&](int&) {
    return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                int(bytes(kMaxSlice, kLocalHist)));
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(a.rows) * unsigned(c));
  cfg.blockDim = dim3(unsigned(threads));
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
