// attn_chunk.cu -- attention of ragged prompt chunks over a KV cache of any layout on the 5th
// generation tensor cores (ATTN for M > 1, src/scripts/lfm-engine/kernels.js:268-319, for several
// sequences at once over paged / int8 / 4-bit caches).
//
// Work.  An item is 256 query rows of one sequence and kv head: 256 / G tokens times the G query
// heads that share the kv head, so that one pass over the keys serves all of them and short chunks
// of grouped heads fill the tensor cores' 128 rows.  An item runs over its keys in tiles of 128.
// All tiles of all items form one list, the longest items of each sequence first, that is cut into
// equal parts, one per SM, so ragged batches and causal prompts balance by themselves and a CTA's
// roles run on from item to item.  An item counts kSetup units more than its tiles, for the start
// and the end of its pipeline (without, the CTAs with a prompt's short first items took 2.5 times
// as long as the others).  An item that straddles CTAs leaves records (unnormalised rows,
// maxima, sums; at most two a CTA, 20 MB in all) which a dependent kernel joins in CTA order.
//
// Roles of a CTA (16 warps, 12 over f16 caches): two softmax warpgroups, one query row per thread,
// 128 rows each; one warp that issues the MMAs; one that issues TMA loads: Q (a 3-D box: the
// group's heads of 128 / G tokens), two items deep, and the cached rows, a box per page: f16 ones
// into the operand tiles, others into a ring (of a 4-bit row the 48 aligned bytes that hold the
// head's 36); four that convert int8 and 4-bit rows, a key per thread, each value rounded to f16
// once, into the swizzled operand layout.  Their loops are rolled: unrolled they took the
// instruction cache from the softmax (16 sequences of 5 tokens: 38 us, 45 unrolled; 4096 4-bit rows
// over 28000 keys: 1720 us, 1785).
//   S_w = Q_w K^T (M128 N128 K64) -> TMEM; P_w to TMEM as f16; O_w += P_w V (M128 N64 K128). The
// softmax: exp2 with the scale folded in, lazily rescaled (only when a row's maximum grows by
// 2^5); the largest weight is put at 2^10, so that as f16 one keeps its bits down to 2^-24 of it and
// is lost below 2^-35 (put at 1, a row over a first key of no value and a tail 17 nats below it was
// 44 % off; the times are the same).  Every fourth pair of exponentials is a cubic on the FMA pipe (4096 f16 rows over 28000
// keys: 1450 us, 1670 with none; the first 5 of 16 pairs in a row: 1628), the others are f32 ones
// rounded once (packed f16 ones round their argument, errors of up to 2^-9 of a weight, and took
// as long); the row sums are taken in f32.
//   A key that a row may not see has weight 0, but 0 * inf and 0 * NaN are NaN: a token whose V
// overflowed would reach the tokens in front of it in its tile.  A row whose sums are not finite
// though it does not see all keys of its tiles is looked at again when the CTA's parts are done,
// and worked out key by key if such a V is the cause.  (Looking through those tiles of V before
// they are multiplied cost 4 prompts of 4096 tokens 384 -> 479 us, this 384 -> 389.)
//
// What bounds it.  Long chunks: a tile's chain in the two softmax warps of each scheduler (4096 rows of
// 32 heads over 28000 keys: 1455 us in f16, 693 TFLOP/s, 1580 us in 4 bits, 638, 1670 us in int8, 604).
// Prompts of up to 4096 tokens: 336 us for four, 576 TFLOP/s of the causal half. Short chunks: latency, 2.3
// us to cut the list, 5 us to the first scores, about 2 us a tile whatever its rows (a warp has a
// row per lane and all 128 keys), 5 us to join (16 sequences of 5 tokens over up to 4096 4-bit
// keys: 40 us).
//
// Every wait is bounded; one that gives up sets the error word, the other roles stop, the CTA frees
// its TMEM and writes nothing more.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "kv_view.cuh"
#include "sm100.cuh"

namespace p2p {
namespace {

using namespace sm100;

constexpr int BM = 128, BN = 128, D = kHeadDim;
constexpr int kRows = 2 * BM;  // rows of an item
constexpr int kMmaWarp = 8, kTmaWarp = 9, kLoadWarp0 = 12, kLoadWarps = 4;
constexpr int kMarks = 16;
constexpr int kSetup = 2;
constexpr int kMinUnits = 3;  // of a CTA: fewer make more records than they save time
constexpr int kStages = 3, kMaxRaw = 2;  // operand tiles; copied rows of int8 and 4-bit caches
constexpr uint32_t kTmemCols = 512;
constexpr uint64_t kWaitLimitNs = 1000000000ull;
// log2 of where a row's largest weight is put, and of how far it may grow before the row is rescaled:
// together below f16's 2^16.
constexpr float kUp = 10.0f, kRescaleLog2 = 5.0f;
// 3 operand tiles, not 4, leave more of the SM to the L1 cache (4 prompts of up to 4096 tokens: 350 us,
// 368 with 4).
// What differs by the cache's format: f16 tiles only move (kMoveF16), int8 and 4-bit rows are copied
// into a ring of kRaw tiles first (4096 4-bit rows over 28000 keys: 2 and 3 of them take as long).
// Registers: setmaxnreg splits what the launch gives (kThreads x kLaunchRegs) among the two softmax
//   warpgroups, that of the issuing warps and that of the converting ones.  The f16 kernel has no
//   converting warps and gives theirs to the others (4 prompts: 350 -> 335 us).  int8: 245 us for 512
//   rows over 32000 keys, 287 with the 4-bit split; 4 bits: 51 us for 512 rows over 3600 keys, 53 with
//   192, 72 and 56.
template <int KVF>
struct Conf {
  static constexpr bool kMoveF16 = KVF == kKvF16;
  static constexpr int kRaw = kMoveF16 ? 0 : kMaxRaw;
  static constexpr int kRowBytes = kMoveF16 ? 128 : KVF == kKvI8 ? 64 : 48;  // of a copied row
  static constexpr int kThreads = kMoveF16 ? 384 : 512, kLaunchRegs = kMoveF16 ? 168 : 128;
  static constexpr int kSoftmaxRegs = KVF == kKvI8 ? 176 : 184,
                       kIssueRegs = kMoveF16 ? 136 : KVF == kKvI8 ? 64 : 72,
                       kLoadRegs = kMoveF16 ? 0 : KVF == kKvI8 ? 96 : 72;
  static_assert(256 * kSoftmaxRegs + 128 * (kIssueRegs + kLoadRegs) <= kThreads * kLaunchRegs,
                "register split");
};
constexpr int kRec = 68;       // a record's row: acc[64], max, sum, 2 pad

__device__ __forceinline__ uint32_t col_s(int w) { return uint32_t(w) * 256u; }
__device__ __forceinline__ uint32_t col_p(int w) { return uint32_t(w) * 256u + 128u; }
__device__ __forceinline__ uint32_t col_o(int w) { return uint32_t(w) * 256u + 192u; }

template <int KVF>
struct __align__(1024) Tiles {
  __half q[2][2][BM * D];   // two items, two halves
  __half kv[kStages][2][BN * D];  // K, V
  unsigned char raw[Conf<KVF>::kRaw ? Conf<KVF>::kRaw : 1][2]
                   [Conf<KVF>::kRaw ? BN * Conf<KVF>::kRowBytes : 16];  // int8, 4 bits: their rows
};
struct __align__(128) Smem {
  float scale[kLoadWarps][2][D];  // int8: the head's scales, a copy per converting warp
  uint64_t q_full[2], q_free[2];
  uint64_t kv_full[kStages], kv_empty[kStages];
  uint64_t raw_full[kMaxRaw], raw_empty[kMaxRaw];
  uint64_t s_full[2], s_free[2], p_full[2], pv_done[2], o_free[2];
  long long wsum[8];
  int z0, qt0, kh0, off0, n_units;  // the first item of the CTA's part, and where in it
  int4 part[8];  // of part i & 7, for the MMA warp: first and end key tile, the halves' tiles
  int part_tail[8];  // its item's keys
  volatile int bad[kMarks];  // of part i % kMarks of this CTA: some page was refused
  volatile int odd;          // some row that does not see all keys of its tiles is not finite
  uint32_t tmem_base;
  volatile int abort_flag;
};

__device__ __forceinline__ bool wait_bar(Smem& s, uint64_t* bar, uint32_t parity, int32_t* err) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if (s.abort_flag) return false;
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      s.abort_flag = 1;
      atomicOr(err, kErrTimeout);
      return false;
    }
  }
}

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// One item: rows of tokens tok0 .. of sequence z for kv head kh.
struct Item {
  int z, kh, qt;
  int past, row0, len;  // of the sequence
  int group;

  __device__ __forceinline__ int tok0() const { return qt * (kRows / group); }
  __device__ __forceinline__ int rows() const { return min(kRows, (len - tok0()) * group); }
  // valid rows of half w, and the keys its last row sees
  __device__ __forceinline__ int rows_of(int w) const { return max(0, min(BM, rows() - BM * w)); }
  __device__ __forceinline__ int key_end(int w) const {
    const int r = rows_of(w);
    return r == 0 ? 0 : past + tok0() + (BM * w + r - 1) / group + 1;
  }
  __device__ __forceinline__ int key_end() const {
    return past + tok0() + (rows() - 1) / group + 1;
  }
  // keys that row r sees
  __device__ __forceinline__ int key_lim(int r) const { return past + tok0() + r / group + 1; }
  __device__ __forceinline__ int tiles() const { return (key_end() + BN - 1) / BN; }
  __device__ __forceinline__ int tiles_of(int w) const { return (key_end(w) + BN - 1) / BN; }
};

__host__ __device__ constexpr int q_tiles(int len, int group) {
  return (len * group + kRows - 1) / kRows;
}
// Key tiles of query tiles 0 .. n - 1 of a sequence: the sum of ceil(keys / 128), where tile q's last
// row sees past + (q + 1) * per keys (`per` a power of two) but the sequence's last tile past + len.
__host__ __device__ inline long long tiles_before(int past, int len, int group, int n) {
  const int per = kRows / group, total = q_tiles(len, group);
  const int full = n == total ? n - 1 : n;  // tiles whose tokens are all there, at least
  long long sum = 0;
  if (full > 0) {
    if (per >= BN) {  // (past + 127) / 128 + q * (per / 128), q = 1 .. full
      const long long a = (static_cast<long long>(past) + BN - 1) / BN;
      sum = a * full + static_cast<long long>(per / BN) * full * (full + 1LL) / 2;
    } else {  // floor((u + q) / k), u = (past + 127) / per, k = 128 / per
      const long long k = BN / per, u = (static_cast<long long>(past) + BN - 1) / per;
      auto upto = [k](long long m) {  // sum over 0 .. m of i / k
        const long long t = m / k;
        return k * (t * (t - 1) / 2) + t * (m - k * t + 1);
      };
      sum = upto(u + full) - upto(u);
    }
  }
  if (full < n) sum += (static_cast<long long>(past) + len + BN - 1) / BN;
  return sum;
}

__host__ __device__ inline long long units_before(int past, int len, int group, int n) {
  return tiles_before(past, len, group, n) + static_cast<long long>(kSetup) * n;
}

// The items in list order: sequences, their query tiles from the last (the longest) to the first,
// the kv heads of each.
struct ItemWalk {
  const KvView& kv;
  const ChunkIndex& at;
  Item it;
  __device__ __forceinline__ ItemWalk(const KvView& k, const ChunkIndex& x, int group, int z,
                                      int qt, int kh)
      : kv(k), at(x) {
    it.group = group;
    it.z = z;
    it.qt = qt;
    it.kh = kh;
    take();
  }
  __device__ __forceinline__ bool take() {
    const SeqSpan sp = seq_span(kv, at, it.z);
    it.past = sp.past;
    it.row0 = sp.row0;
    it.len = sp.ok ? sp.len : 0;
    return it.len > 0;
  }
  __device__ __forceinline__ void next() {
    if (++it.kh < kv.hkv) return;
    it.kh = 0;
    if (--it.qt >= 0) return;
    do ++it.z;
    while (it.z < at.nseq && !take());
    it.qt = q_tiles(it.len, it.group) - 1;
  }
};

// A CTA's parts of items, one after the other: the key tiles k0 .. k1 - 1 of each.
struct PartWalk {
  ItemWalk walk;
  int off, left;  // unit of the item where the part begins, units of the CTA from there
  int nk, k0, k1, seg;
  bool live;
  __device__ __forceinline__ PartWalk(const KvView& k, const ChunkIndex& x, int group,
                                      const Smem& s)
      : walk(k, x, group, s.z0, s.qt0, s.kh0), off(s.off0), left(s.n_units), seg(0) {
    set();
  }
  __device__ __forceinline__ void set() {
    nk = walk.it.tiles();
    k0 = max(0, off - kSetup);
    k1 = min(nk, off + left - kSetup);
    live = k1 > k0;  // a CTA's units may end before the item's first tile
  }
  __device__ __forceinline__ void next() {
    left -= kSetup + nk - off;
    off = 0;
    ++seg;
    live = false;
    if (left <= 0) return;
    walk.next();
    set();
  }
  __device__ __forceinline__ const Item& it() const { return walk.it; }
};
// Their tiles, one after the other.
struct TileStream {
  PartWalk part;
  int jj;
  __device__ __forceinline__ TileStream(const KvView& k, const ChunkIndex& x, int group,
                                        const Smem& s)
      : part(k, x, group, s), jj(part.k0) {}
  __device__ __forceinline__ bool done() const { return !part.live; }
  __device__ __forceinline__ void next() {
    if (++jj < part.k1) return;
    part.next();
    jj = part.k0;
  }
  __device__ __forceinline__ const Item& it() const { return part.walk.it; }
  __device__ __forceinline__ int valid() const { return min(BN, it().key_end() - jj * BN); }
};

// Eight 4-bit codes of a word as f16 values code * s + lo (one rounding: an f16 multiply-add).
__device__ __forceinline__ uint4 q4_piece(uint32_t w, uint32_t params) {
  const uint32_t s2 = __byte_perm(params, params, 0x1010), l2 = __byte_perm(params, params, 0x3232);
  const __half2 s = *reinterpret_cast<const __half2*>(&s2);
  const __half2 lo = *reinterpret_cast<const __half2*>(&l2);
  const __half2 base = __floats2half2_rn(1024.f, 1024.f);
  uint32_t r[4];  // values i and i + 4
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t c = ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u;  // 1024 + code
    const __half2 v = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&c), base), s, lo);
    r[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(__byte_perm(r[0], r[1], 0x5410), __byte_perm(r[2], r[3], 0x5410),
                    __byte_perm(r[0], r[1], 0x7632), __byte_perm(r[2], r[3], 0x7632));
}

// Bytes 2k, 2k + 1 of x ^ 0x80808080 (x: signed bytes) times their scales, rounded to f16 once: under
// the f32 pattern of 2^23 a byte is 2^23 + 128 + its value (no conversion instructions, which would
// share the exponentials' unit).
__device__ __forceinline__ uint32_t s8_scaled(uint32_t w, int k, float s0, float s1) {
  const float f0 = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + 2 * k));
  const float f1 = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441 + 2 * k));
  uint64_t x, s;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(f0), "f"(f1));
  asm("mov.b64 %0, {%1, %2};" : "=l"(s) : "f"(s0), "f"(s1));
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(0xcb000080cb000080ull));  // -(2^23 + 128)
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(s));
  float v0, v1;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v0), "=f"(v1) : "l"(x));
  return pack_half2(v0, v1);
}

// The maximum of three, NaN when one of them is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// acc += (a, b), a pair of f32 sums; and their total.
__device__ __forceinline__ void add_pair(uint64_t& acc, float a, float b) {
  uint64_t x;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a), "f"(b));
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(acc) : "l"(x));
}
__device__ __forceinline__ float pair_sum(uint64_t acc) {
  float a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(acc));
  return a + b;
}

// Dims 8 i .. 8 i + 7 of a cached row as the MMAs see them.
__device__ __forceinline__ void cached_piece(const KvView& kv, int pool, int64_t row, int kh, int i,
                                             float (&x)[8]) {
  const unsigned char* src = (pool ? kv.v : kv.k) + row * kv.row_bytes;
  uint4 h;
  if (kv.format == kKvF16) {
    h = reinterpret_cast<const uint4*>(src + kh * 128)[i];
  } else if (kv.format == kKvQ4) {
    const uint32_t* unit = reinterpret_cast<const uint32_t*>(src + kh * kQ4UnitBytes);
    h = q4_piece(unit[i], unit[8]);
  } else {
    const float* sc = pool ? kv.v_scale : kv.k_scale;
    float v[8];
    for (int k = 0; k < 8; ++k)
      v[k] = float(reinterpret_cast<const int8_t*>(src)[kh * D + 8 * i + k]) *
             sc[kv.per_channel ? kh * D + 8 * i + k : 0];
    h = make_uint4(pack_half2(v[0], v[1]), pack_half2(v[2], v[3]), pack_half2(v[4], v[5]),
                   pack_half2(v[6], v[7]));
  }
  const uint32_t w[4] = {h.x, h.y, h.z, h.w};
  for (int k = 0; k < 4; ++k) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
    x[2 * k] = f.x;
    x[2 * k + 1] = f.y;
  }
}

// Row r of an item over the keys k0 .. k1 - 1 of its tiles, of which it sees those below its limit:
// if a V behind the limit is not finite, the row is worked out again without it, into the f16
// output or the f32 record that the calling thread wrote before.
__device__ __noinline__ void redo_row(const ChunkArgs& a, const Item& it, int r, int k0, int k1,
                                      __half* out, float* rec) {
  const int lim = min(k1, it.key_lim(r));
  float x[8], acc[D], m = -INFINITY, l = 0.f;
  bool odd = false;
  for (int key = max(k0, it.key_lim(r)); key < k1; ++key) {
    const int64_t row = kv_row(a.kv, it.z, key);
    if (row < 0) return;  // refused: the row was not written
    for (int i = 0; i < 8; ++i) {
      cached_piece(a.kv, 1, row, it.kh, i, x);
      for (int k = 0; k < 8; ++k) odd |= !(fabsf(x[k]) < INFINITY);
    }
  }
  if (!odd) return;
  const __half* q = a.q + (int64_t(it.row0) + it.tok0() + r / it.group) * a.ld_q +
                    (it.kh * it.group + r % it.group) * D;
  for (int d = 0; d < D; ++d) acc[d] = 0.f;
  for (int key = k0; key < lim; ++key) {
    const int64_t row = kv_row(a.kv, it.z, key);
    if (row < 0) return;
    float sc = 0.f;
    for (int i = 0; i < 8; ++i) {
      cached_piece(a.kv, 0, row, it.kh, i, x);
      for (int k = 0; k < 8; ++k) sc = fmaf(__half2float(q[8 * i + k]), x[k], sc);
    }
    sc *= a.scale_log2;
    if (sc == -INFINITY) continue;
    if (sc > m) {
      const float c = fast_exp2(m - sc);
      m = sc;
      l *= c;
      for (int d = 0; d < D; ++d) acc[d] *= c;
    }
    const float p = fast_exp2(sc - m);
    l += p;
    for (int i = 0; i < 8; ++i) {
      cached_piece(a.kv, 1, row, it.kh, i, x);
      for (int k = 0; k < 8; ++k) acc[8 * i + k] = fmaf(p, x[k], acc[8 * i + k]);
    }
  }
  if (out) {
    const float inv = __fdiv_rn(1.0f, l);
    for (int d = 0; d < D; ++d) out[d] = __float2half_rn(acc[d] * inv);
  } else {
    for (int d = 0; d < D; ++d) rec[d] = acc[d];
    rec[D] = m == -INFINITY ? -1e30f : m;
    rec[D + 1] = l;
  }
}

template <int KVF>
__global__ void __launch_bounds__(Conf<KVF>::kThreads, 1)
    attn_chunk_kernel(const __grid_constant__ CUtensorMap tm_q,
                      const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ ChunkArgs a) {
  extern __shared__ uint8_t smem_raw[];
  constexpr bool kMoveF16 = Conf<KVF>::kMoveF16;
  auto& tiles = *reinterpret_cast<Tiles<KVF>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Smem& s = *reinterpret_cast<Smem*>(&tiles + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = a.hq / a.kv.hkv, gshift = __ffs(group) - 1;

  // ---- this CTA's part of the list
  const int per = (a.at.nseq + 255) / 256;
  long long mine = 0, upto = 0, total = 0;
  if (tid < 256) {
    for (int z = tid * per; z < min((tid + 1) * per, a.at.nseq); ++z) {
      const SeqSpan sp = seq_span(a.kv, a.at, z);
      if (!sp.ok) {
        if (blockIdx.x == 0) atomicOr(a.err, kErrPosBeyondCache);
      } else if (sp.len > 0) {
        mine += a.kv.hkv * units_before(sp.past, sp.len, group, q_tiles(sp.len, group));
      }
    }
    upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) s.wsum[warp] = upto;
  }
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.kv_full[i], KVF == kKvF16 ? 1 : kLoadWarps);
      mbar_init(&s.kv_empty[i], 1);
    }
    for (int i = 0; i < Conf<KVF>::kRaw; ++i) {
      mbar_init(&s.raw_full[i], 1);
      mbar_init(&s.raw_empty[i], kLoadWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.q_full[i], 1);
      mbar_init(&s.q_free[i], 1);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.s_free[i], 4);
      mbar_init(&s.p_full[i], 4);
      mbar_init(&s.pv_done[i], 1);
      mbar_init(&s.o_free[i], 4);
    }
    for (int i = 0; i < kMarks; ++i) s.bad[i] = 0;
    s.odd = 0;
    s.abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    if (w == warp) upto += total;
    total += s.wsum[w];
  }
  const int parts = int(min(static_cast<long long>(gridDim.x),
                            (total + kMinUnits - 1) / kMinUnits));
  const int b = blockIdx.x;
  launch_dependents();
  if (tid == 0) a.joins[b] = make_int4(-1, 0, 0, 0);
  if (b >= parts) return;
  const long long lo = total * b / parts;
  if (tid < 256 && lo < upto && lo >= upto - mine) {
    long long at = upto - mine;
    for (int z = tid * per;; ++z) {
      const SeqSpan sp = seq_span(a.kv, a.at, z);
      if (!sp.ok || sp.len <= 0) continue;
      const int nq = q_tiles(sp.len, group);
      const long long all = units_before(sp.past, sp.len, group, nq);
      const long long r = lo - at;  // the sequence's query tiles come last one first
      at += all * a.kv.hkv;
      if (lo >= at) continue;
      int first = 0, last = nq - 1;  // the tile qt with after(qt) <= r < after(qt - 1)
      auto after = [&](int qt) {
        return (all - units_before(sp.past, sp.len, group, qt + 1)) * a.kv.hkv;
      };
      while (first < last) {
        const int mid = (first + last) / 2;
        if (after(mid) <= r) last = mid;
        else first = mid + 1;
      }
      const int unit = Item{z, 0, first, sp.past, sp.row0, sp.len, group}.tiles() + kSetup;
      const long long in = r - after(first);
      s.z0 = z;
      s.qt0 = first;
      s.kh0 = int(in / unit);
      s.off0 = int(in % unit);
      s.n_units = int(total * (b + 1) / parts - lo);
      break;
    }
  }
  if (warp == kMmaWarp) tmem_alloc(&s.tmem_base, kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem_base;
  const int n_units = s.n_units;

  if (!kMoveF16 && warp >= kLoadWarp0) {
    if constexpr (!kMoveF16) regs_dec<Conf<KVF>::kLoadRegs>();
    // ---------------------------------------------------------------- converting warps
    constexpr int kRaw = Conf<KVF>::kRaw ? Conf<KVF>::kRaw : 1, kRowBytes = Conf<KVF>::kRowBytes;
    const int key = tid - kLoadWarp0 * 32;
    TileStream tile(a.kv, a.at, group, s);
    int head = -1, st = 0, rs = 0;
    uint32_t ph = 1, rph = 0;
    for (int c = 0; !tile.done(); ++c, tile.next()) {
      const int kh = tile.it().kh;
      const bool there = key < tile.valid();  // rows behind the last key: zeros
      bool ok = wait_bar(s, &s.raw_full[rs], rph, a.err);
      if (ok && c >= kStages) ok = wait_bar(s, &s.kv_empty[st], ph, a.err);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (KVF == kKvI8 && kh != head) {
        __syncwarp();
#pragma unroll
        for (int pool = 0; pool < 2; ++pool)
#pragma unroll
          for (int d = lane; d < D; d += 32)
            s.scale[warp - kLoadWarp0][pool][d] =
                (pool ? a.kv.v_scale : a.kv.k_scale)[a.kv.per_channel ? kh * D + d : 0];
        __syncwarp();
        head = kh;
      }
#pragma unroll 1
      for (int pool = 0; pool < 2; ++pool) {
        const unsigned char* src = &tiles.raw[rs][pool][key * kRowBytes];
        char* dst = reinterpret_cast<char*>(tiles.kv[st][pool]) + key * 128;
        if constexpr (KVF == kKvQ4) {
          // the unit's 9 words among the 12 that were copied
          const uint32_t* unit = reinterpret_cast<const uint32_t*>(src) + (kh & 3);
          const uint32_t params = there ? unit[8] : 0u;
#pragma unroll 2
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint4*>(dst + ((i ^ (key & 7)) << 4)) =
                q4_piece(there ? unit[i] : 0u, params);
        } else {
          const float4* scale = reinterpret_cast<const float4*>(s.scale[warp - kLoadWarp0][pool]);
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {  // 16-byte pieces, swizzled over 8 rows by the copy
            const uint4 w =
                there ? *reinterpret_cast<const uint4*>(src + ((i ^ ((key >> 1) & 3)) << 4))
                      : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float4 lo = scale[4 * i + 2 * k], hi = scale[4 * i + 2 * k + 1];
              const uint32_t w0 = (k ? w.z : w.x) ^ 0x80808080u, w1 = (k ? w.w : w.y) ^ 0x80808080u;
              *reinterpret_cast<uint4*>(dst + (((2 * i + k) ^ (key & 7)) << 4)) =
                  make_uint4(s8_scaled(w0, 0, lo.x, lo.y), s8_scaled(w0, 1, lo.z, lo.w),
                             s8_scaled(w1, 0, hi.x, hi.y), s8_scaled(w1, 1, hi.z, hi.w));
            }
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&s.raw_empty[rs]);
        mbar_arrive(&s.kv_full[st]);
      }
      if (++st == kStages) {
        st = 0;
        ph ^= 1;
      }
      if (++rs == kRaw) {
        rs = 0;
        rph ^= 1;
      }
    }
  } else if (warp >= 8) {
    regs_dec<Conf<KVF>::kIssueRegs>();
    if (warp == kMmaWarp) {
      // ---------------------------------------------------------------- MMA issuer
      constexpr uint32_t idesc_s = idesc_f16_f32(BM, BN, 0, 0);
      constexpr uint32_t idesc_pv = idesc_f16_f32(BM, D, 0, 1);
      static_assert(sizeof(tiles.q[0]) == 32768 && sizeof(tiles.kv[0]) == 32768, "16 KB tiles");
      const uint64_t qdesc0 = smem_desc_sw128(smem_u32(tiles.q[0][0]), 16, 1024);
      const uint64_t kdesc0 = smem_desc_sw128(smem_u32(tiles.kv[0][0]), 16, 1024);
      const uint64_t vdesc0 = smem_desc_sw128(smem_u32(tiles.kv[0][1]), 0, 1024);
      uint32_t seg = 0;  // parts so far
      auto issue_s = [&](int w, int st) {  // S_w = Q_w K_st^T
        if (elect_one()) {
          const uint64_t qd = qdesc0 + uint64_t((seg & 1) * 2 + w) * 1024,
                         kd = kdesc0 + uint64_t(st) * 2048;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            mma_f16_ss(tmem + col_s(w), qd + 2 * kk, kd + 2 * kk, idesc_s, kk > 0);
          mma_commit(&s.s_full[w]);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int w, int st, bool acc) {  // O_w += P_w V_st
        if (elect_one()) {
          const uint64_t vd = vdesc0 + uint64_t(st) * 2048;
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            mma_f16_ts(tmem + col_o(w), tmem + col_p(w) + kk * 8, vd + 128 * kk, idesc_pv,
                       (acc || kk > 0) ? 1u : 0u);
          mma_commit(&s.pv_done[w]);
        }
        __syncwarp();
      };
      auto wait_warp = [&](uint64_t* bar, uint32_t parity) {
        bool r = true;
        if (lane == 0) r = wait_bar(s, bar, parity, a.err);
        return __shfl_sync(0xffffffffu, r ? 1 : 0, 0) != 0;
      };
      int st = 0, st1 = 1 % kStages;       // stage of this tile and of the next
      uint32_t ph = 0, ph1 = 0;            // their parities
      uint32_t n_s0 = 0, n_s1 = 0, n_pv0 = 0, n_pv1 = 0, n_o0 = 0, n_o1 = 0;  // per half: S, P.V,
      bool ok = true;                                                         // ended O
      while (ok) {
        ok = wait_warp(&s.q_full[seg & 1], (seg >> 1) & 1);
        if (!ok) break;
        const int4 part = s.part[seg & 7];
        const int k1 = part.y, nk0 = part.z, nk1 = part.w;
        if (k1 == 0) break;  // behind the last part
        // S of both halves for key tile jj in stage x, where they have rows that see it
        auto score = [&](int jj, int x) {
          if (jj < nk0) {
            if (n_s0 > 0 && !wait_warp(&s.s_free[0], (n_s0 - 1) & 1)) return false;
            tc_fence_after();
            issue_s(0, x);
            ++n_s0;
          }
          if (jj < nk1) {
            if (n_s1 > 0 && !wait_warp(&s.s_free[1], (n_s1 - 1) & 1)) return false;
            tc_fence_after();
            issue_s(1, x);
            ++n_s1;
          }
          return true;
        };
        ok = wait_warp(&s.kv_full[st], ph);
        tc_fence_after();
        ok = ok && score(part.x, st);
        for (int jj = part.x; ok && jj < k1; ++jj) {
          if (jj + 1 < k1) {  // the next tile's scores, while the softmax of this one runs
            ok = wait_warp(&s.kv_full[st1], ph1);
            tc_fence_after();
            ok = ok && score(jj + 1, st1);
            if (!ok) break;
          } else {
            if (elect_one()) mma_commit(&s.q_free[seg & 1]);
            __syncwarp();
            const int tail = s.part_tail[seg & 7] - jj * BN;
            if (KVF == kKvF16 && tail < BN) {
              // Rows behind the last key may hold anything; P is 0 there, but 0 * NaN is NaN
              uint4* vrow = reinterpret_cast<uint4*>(tiles.kv[st][1]);
              for (int i = tail * 8 + lane; i < BN * 8; i += 32) vrow[i] = make_uint4(0, 0, 0, 0);
              fence_proxy_async_smem();
              __syncwarp();
            }
          }
          if (jj < nk0) {
            if (jj == part.x && n_o0 > 0) ok = wait_warp(&s.o_free[0], (n_o0 - 1) & 1);
            ok = ok && wait_warp(&s.p_full[0], n_pv0 & 1);
            if (!ok) break;
            tc_fence_after();
            issue_pv(0, st, jj > part.x);
            ++n_pv0;
          }
          if (jj < nk1) {
            if (jj == part.x && n_o1 > 0) ok = wait_warp(&s.o_free[1], (n_o1 - 1) & 1);
            ok = ok && wait_warp(&s.p_full[1], n_pv1 & 1);
            if (!ok) break;
            tc_fence_after();
            issue_pv(1, st, jj > part.x);
            ++n_pv1;
          }
          if (elect_one()) mma_commit(&s.kv_empty[st]);
          __syncwarp();
          st = st1;
          ph = ph1;
          if (++st1 == kStages) {
            st1 = 0;
            ph1 ^= 1;
          }
        }
        if (part.x < nk0) ++n_o0;
        if (part.x < nk1) ++n_o1;
        ++seg;
      }
    } else if (warp == kTmaWarp) {
      // ---------------------------------------------------------------- TMA producer
      // f16 rows go straight to the operand tiles, others to the ring of the converting warps
      constexpr int kRing = kMoveF16 ? kStages : Conf<KVF>::kRaw, kRowBytes = Conf<KVF>::kRowBytes;
      uint64_t* full = kMoveF16 ? s.kv_full : s.raw_full;
      uint64_t* empty = kMoveF16 ? s.kv_empty : s.raw_empty;
      unsigned char* ring =
          kMoveF16 ? reinterpret_cast<unsigned char*>(tiles.kv) : &tiles.raw[0][0][0];
      const bool paged = a.kv.table != nullptr;
      const int mask = (1 << a.kv.shift) - 1;
      PartWalk walk(a.kv, a.at, group, s);
      int c = 0, n_q = 0;
      bool ok = true;
      if (lane == 0) {
        prefetch_tensormap(&tm_q);
        prefetch_tensormap(&tm_k);
        prefetch_tensormap(&tm_v);
      }
      for (bool more = true; more; walk.next()) {
        const Item it = walk.it();
        const int seg = walk.seg, k0 = walk.k0, k1 = walk.k1, key_end = it.key_end();
        more = walk.live;
        // Q (and what the MMA warp has to know) once the products of two items before are done
        if (seg > 1) {
          if (lane == 0) ok = wait_bar(s, &s.q_free[seg & 1], ((seg >> 1) - 1) & 1, a.err);
          ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
          if (!ok) break;
        }
        if (!more) {  // tells the MMA warp that the part before was the last
          if (lane == 0) {
            s.part[seg & 7] = make_int4(0, 0, 0, 0);
            mbar_arrive(&s.q_full[seg & 1]);
          }
          break;
        }
        if (lane == 0) {
          // The mark of eight parts ahead is cleared.  The part that used it last is eight back,
          // and ended long ago.
          s.bad[(seg + kMarks / 2) % kMarks] = 0;
          s.part[seg & 7] = make_int4(k0, k1, it.tiles_of(0), it.tiles_of(1));
          s.part_tail[seg & 7] = key_end;
          const int halves = it.rows() > BM ? 2 : 1;
          mbar_arrive_expect_tx(&s.q_full[seg & 1], uint32_t(halves * BM * D * 2));
          for (int h = 0; h < halves; ++h)
            tma_load_3d(tiles.q[seg & 1][h], &tm_q, 0, it.kh * group,
                        it.row0 + it.tok0() + h * (BM >> gshift), &s.q_full[seg & 1]);
        }
        n_q = seg + 1;
        const int x = KVF == kKvQ4 ? it.kh * kQ4UnitBytes / 16 * 16 : it.kh * D;
        int32_t pages = 0;
        const int off = paged ? 0 : a.kv.offsets[it.z];
        for (int jj = k0; jj < k1; ++jj, ++c) {
          const int st = c % kRing, key0 = jj * BN, valid = min(BN, key_end - key0);
          if (lane == 0 && c >= kRing)
            ok = wait_bar(s, &empty[st], (c / kRing - 1) & 1, a.err);
          ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
          if (!ok) break;
          // one box per page (or one of 128 rows)
          const int box = paged ? min(1 << a.kv.shift, BN) : BN;
          const int boxes = (valid + box - 1) / box;
          int64_t row = int64_t(off) + key0;
          if (paged) {
            const int in = (jj - k0) & 3;  // the pages of four tiles at a time, at most 32
            if (in == 0) {
              pages = 0;
              const int p = (key0 >> a.kv.shift) + lane;
              if (p <= (key_end - 1) >> a.kv.shift)
                pages = a.kv.table[int64_t(it.z) * a.kv.max_blocks + p];
            }
            const int at = key0 + min(lane, boxes - 1) * box;
            const int32_t pg = __shfl_sync(
                0xffffffffu, pages, (at >> a.kv.shift) - ((key0 - in * BN) >> a.kv.shift));
            row = pg < 0 || int64_t(pg) >= a.kv.kv_rows
                      ? -1
                      : (int64_t(pg) << a.kv.shift) | (at & mask);
          }
          const bool bad = __any_sync(0xffffffffu, row < 0);
          if (lane == 0) {
            if (bad) {
              s.bad[seg % kMarks] = 1;
              atomicOr(a.err, kErrPosBeyondCache);
            }
            mbar_arrive_expect_tx(&full[st],
                                  uint32_t(bad ? 0 : 2 * boxes * box * kRowBytes) +
                                      uint32_t(c == 0 ? a.wait_deficit : 0));
          }
          __syncwarp();
          if (!bad && lane < boxes) {
            unsigned char* dst = ring + st * 2 * BN * kRowBytes + lane * box * kRowBytes;
            tma_load_2d(dst, &tm_k, x, int32_t(row), &full[st]);
            tma_load_2d(dst + BN * kRowBytes, &tm_v, x, int32_t(row), &full[st]);
          }
        }
        if (!ok) break;
      }
      // after a wait that ran out: let the copies already in flight land before the CTA exits
      if (lane == 0 && s.abort_flag) {
        const uint64_t t0 = globaltimer_ns();
        for (int i = max(0, n_q - 2); i < n_q; ++i)
          while (!mbar_try_wait(&s.q_full[i & 1], (i >> 1) & 1) &&
                 globaltimer_ns() - t0 < kWaitLimitNs) {
          }
        for (int i = max(0, c - kRing); i < c; ++i)
          while (!mbar_try_wait(&full[i % kRing], (i / kRing) & 1) &&
                 globaltimer_ns() - t0 < kWaitLimitNs) {
          }
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax warpgroups
    regs_inc<Conf<KVF>::kSoftmaxRegs>();
    const int w = warp >> 2;
    const int r = tid & 127;  // row of the half = TMEM lane
    const uint32_t lane_addr = tmem + (uint32_t((warp & 3) * 32) << 16);
    const float sl2 = a.scale_log2;
    PartWalk walk(a.kv, a.at, group, s);
    int n = 0;  // tiles of this half
    bool ok = true;
    for (; walk.live; walk.next()) {
      const Item it = walk.it();
      const int seg = walk.seg, nk = walk.nk, k0 = walk.k0, k1 = walk.k1;
      const int rows = it.rows_of(w), mine_end = min(k1, it.tiles_of(w));
      if (rows == 0) continue;
      const int first_lim = it.key_lim(BM * w);  // keys the first row sees
      const int key_lim = first_lim + r / group;
      float m_raw = -INFINITY, l_run = 0.f;
      for (int j = k0; j < mine_end; ++j, ++n) {
        ok = wait_bar(s, &s.s_full[w], n & 1, a.err);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t sv[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(lane_addr + col_s(w) + q * 32, sv[q]);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.s_free[w]);
        const int key0 = j * BN;
        if (key0 + BN > first_lim) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (key0 + q * 32 + i >= key_lim) sv[q][i] = __float_as_uint(-INFINITY);
        }
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            m4[(i >> 1) & 3] = max3_nan(m4[(i >> 1) & 3], __uint_as_float(sv[q][i]),
                                        __uint_as_float(sv[q][i + 1]));
        const float mx = max3_nan(m4[0], max3_nan(m4[1], m4[1], m4[2]), m4[3]);
        const bool grow = (mx - m_raw) * sl2 > kRescaleLog2;
        const float alpha = grow ? fast_exp2((m_raw - mx) * sl2) : 1.0f;
        if (grow) m_raw = mx;
        // a score of NaN or +inf makes all of the row's weights NaN (inf - inf is NaN for that key
        // alone, and the cubic would lose it)
        const float neg = !(mx < INFINITY) ? NAN : (m_raw == -INFINITY) ? 0.f : kUp - m_raw * sl2;
        uint32_t pk[2][32];
        uint64_t ps[4] = {0, 0, 0, 0};  // f32 pairs
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            const int q = half * 2 + cc;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float x0, x1;
              fma2(__uint_as_float(sv[q][2 * i]), __uint_as_float(sv[q][2 * i + 1]), sl2, neg, x0,
                   x1);
              if ((i & 3) == 0) {
                ex2_poly(x0, x1);
              } else {
                x0 = fast_exp2(x0);
                x1 = fast_exp2(x1);
              }
              add_pair(ps[i & 3], x0, x1);
              pk[half][cc * 16 + i] = pack_half2(x0, x1);
            }
          }
        const float sum = (pair_sum(ps[0]) + pair_sum(ps[1])) + (pair_sum(ps[2]) + pair_sum(ps[3]));
        // P is free (and O holds the tiles before) once the last P.V has completed
        if (j > k0) {
          ok = wait_bar(s, &s.pv_done[w], (n - 1) & 1, a.err);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
        }
        tc_fence_after();
        tmem_st32(lane_addr + col_p(w), pk[0]);
        tmem_st32(lane_addr + col_p(w) + 32, pk[1]);
        tmem_st_wait();
        l_run = fmaf(l_run, alpha, sum);
        if (j > k0 && __any_sync(0xffffffffu, grow)) {
          uint32_t ov[2][32];
          tmem_ld32(lane_addr + col_o(w), ov[0]);
          tmem_ld32(lane_addr + col_o(w) + 32, ov[1]);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            ov[0][i] = __float_as_uint(__uint_as_float(ov[0][i]) * alpha);
            ov[1][i] = __float_as_uint(__uint_as_float(ov[1][i]) * alpha);
          }
          tmem_st32(lane_addr + col_o(w), ov[0]);
          tmem_st32(lane_addr + col_o(w) + 32, ov[1]);
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full[w]);
      }
      if (!ok) break;
      const bool whole = k0 == 0 && k1 == nk;
      uint32_t ov[2][32];
      if (k0 < mine_end) {
        ok = wait_bar(s, &s.pv_done[w], (n - 1) & 1, a.err);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        tmem_ld32(lane_addr + col_o(w), ov[0]);
        tmem_ld32(lane_addr + col_o(w) + 32, ov[1]);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.o_free[w]);
        if (mine_end * BN > first_lim) {  // some row does not see all keys of its tiles
          float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < 64; ++i) t[i & 3] += __uint_as_float(ov[i >> 5][i & 31]);
          const float sum = (t[0] + t[1]) + (t[2] + t[3]);
          if (!(fabsf(sum) < INFINITY) && r < rows) s.odd = 1;
        }
      } else {  // this half's keys all lie in other CTAs' parts
#pragma unroll
        for (int i = 0; i < 32; ++i) ov[0][i] = ov[1][i] = 0u;
      }
      // No key that counts so far (scores of -inf, or none in this part): the cubic has left 2^-125 per
      // masked key.  With 0 the row is NaN if that stays all of it, and a record adds nothing.
      if (m_raw == -INFINITY) l_run *= 0.f;
      const bool bad = s.bad[seg % kMarks] != 0;
      if (!whole && tid == 0 && k0 == 0) {  // the item begins here: what there is to join
        // list position behind the item
        const long long end = lo + (n_units - walk.left) - walk.off + kSetup + nk;
        const int last = int((end * parts - 1) / total);
        a.joins[b] = make_int4(it.z, it.kh, it.qt, ((last - b + 1) << 1) | (seg == 0 ? 0 : 1));
      }
      if (r < rows) {
        if (whole) {
          if (!bad) {
            const float inv = __fdiv_rn(1.0f, l_run);
            uint4* dst = reinterpret_cast<uint4*>(
                a.out + (int64_t(it.row0) + it.tok0() + (BM * w + r) / group) * a.ld_o +
                (it.kh * group + r % group) * D);
#pragma unroll
            for (int i = 0; i < D; i += 8) {
              const uint32_t* o = &ov[i >> 5][i & 31];
              dst[i / 8] = make_uint4(
                  pack_half2(__uint_as_float(o[0]) * inv, __uint_as_float(o[1]) * inv),
                  pack_half2(__uint_as_float(o[2]) * inv, __uint_as_float(o[3]) * inv),
                  pack_half2(__uint_as_float(o[4]) * inv, __uint_as_float(o[5]) * inv),
                  pack_half2(__uint_as_float(o[6]) * inv, __uint_as_float(o[7]) * inv));
            }
          }
        } else {
          float4* rec = reinterpret_cast<float4*>(
              a.parts + ((int64_t(b) * 2 + (seg == 0 ? 0 : 1)) * kRows + BM * w + r) * kRec);
#pragma unroll
          for (int i = 0; i < D; i += 4) {
            const uint32_t* o = &ov[i >> 5][i & 31];
            rec[i / 4] = make_float4(__uint_as_float(o[0]), __uint_as_float(o[1]),
                                     __uint_as_float(o[2]), __uint_as_float(o[3]));
          }
          // log2 units; a sum below 0: some page was refused
          const float m2 = m_raw == -INFINITY ? -1e30f : m_raw * sl2 - kUp;
          rec[16] = make_float4(m2, bad ? -1.f : l_run, 0.f, 0.f);
        }
      }
    }
    // a wait ran out: a part that others join is marked, the rest stays as it was
    if (!ok) {
      PartWalk again(a.kv, a.at, group, s);
      for (; again.live; again.next()) {
        const int i = again.seg;
        if (i < walk.seg || (again.k0 == 0 && again.k1 == again.nk) ||
            r >= again.it().rows_of(w))
          continue;
        float* rec = a.parts + ((int64_t(b) * 2 + (i == 0 ? 0 : 1)) * kRows + BM * w + r) * kRec;
        rec[64] = -1e30f;
        rec[65] = -1.f;
      }
    } else if (s.odd) {
      PartWalk again(a.kv, a.at, group, s);
      for (; again.live; again.next()) {
        const Item it = again.it();
        const int row = BM * w + r, first = again.k0 * BN;
        const int end = min(min(again.k1, it.tiles_of(w)) * BN, it.key_end());
        if (row >= it.rows() || end <= it.key_lim(row) || end <= first) continue;
        const bool whole = again.k0 == 0 && again.k1 == again.nk;
        __half* out = a.out + (int64_t(it.row0) + it.tok0() + row / group) * a.ld_o +
                      (it.kh * group + row % group) * D;
        float* rec = a.parts +
                     ((int64_t(b) * 2 + (again.seg == 0 ? 0 : 1)) * kRows + row) * kRec;
        bool finite = true;
        for (int d = 0; d < D; ++d)
          finite = finite && fabsf(whole ? __half2float(out[d]) : rec[d]) < INFINITY;
        if (finite || (!whole && rec[D + 1] < 0.f)) continue;  // < 0: a page was refused
        redo_row(a, it, row, first, end, whole ? out : nullptr, rec);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// CTA (b, y): rows 32 y .. of the item that began in CTA b and went on in others.  Half a warp per
// row (16 lanes of 4 dims), records in CTA order, eight of them in flight.
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads, 4)
    join_chunk_kernel(const __grid_constant__ ChunkArgs a) {
  grid_dependency_wait();
  const int4 d = a.joins[blockIdx.x];
  if (d.x < 0) return;
  const int group = a.hq / a.kv.hkv, b = blockIdx.x, n = d.w >> 1, slot = d.w & 1;
  const SeqSpan sp = seq_span(a.kv, a.at, d.x);
  const Item it{d.x, d.y, d.z, sp.past, sp.row0, sp.len, group};
  const int l16 = threadIdx.x & 15, end = min(it.rows(), int(blockIdx.y) * 32 + 32);
#pragma unroll 1
  for (int r = blockIdx.y * 32 + (threadIdx.x >> 4); r < end; r += 16) {
    auto rec = [&](int i) {
      return a.parts + ((int64_t(b + i) * 2 + (i == 0 ? slot : 0)) * kRows + r) * kRec;
    };
    float mx = -1e30f, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    bool bad = false;
    for (int i0 = 0; i0 < n; i0 += 8) {
      float2 ml[8];
      float4 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float* p = rec(min(i0 + i, n - 1));
        ml[i] = __ldcg(reinterpret_cast<const float2*>(p + 64));
        x[i] = __ldcg(reinterpret_cast<const float4*>(p) + l16);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i0 + i >= n) continue;
        bad |= ml[i].y < 0.f;
        const float m = fmaxf(mx, ml[i].x), c = fast_exp2(mx - m), w = fast_exp2(ml[i].x - m);
        mx = m;
        l = fmaf(l, c, ml[i].y * w);
        acc.x = fmaf(acc.x, c, x[i].x * w);
        acc.y = fmaf(acc.y, c, x[i].y * w);
        acc.z = fmaf(acc.z, c, x[i].z * w);
        acc.w = fmaf(acc.w, c, x[i].w * w);
      }
    }
    if (bad) continue;
    const float inv = __fdiv_rn(1.f, l);
    reinterpret_cast<uint2*>(a.out + (int64_t(it.row0) + it.tok0() + r / group) * a.ld_o +
                             (it.kh * group + r % group) * D)[l16] =
        make_uint2(pack_half2(acc.x * inv, acc.y * inv), pack_half2(acc.z * inv, acc.w * inv));
  }
}

PFN_cuTensorMapEncodeTiled_v12000 get_encode() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// A pool as [rows][the row's values], boxes of one head x `box_rows` rows: f16 in the operands' swizzle,
// int8 in one without bank conflicts for a row per lane; 4 bits as the 48 bytes that hold a unit.
bool make_map(CUtensorMap* m, const void* base, const KvView& kv, int64_t rows, int box_rows) {
  auto enc = get_encode();
  if (!enc) return false;
  const bool f16 = kv.format == kKvF16;
  cuuint64_t dims[2] = {cuuint64_t(f16 ? kv.row_bytes / 2 : kv.row_bytes), cuuint64_t(rows)};
  cuuint64_t strides[1] = {cuuint64_t(kv.row_bytes)};
  cuuint32_t box[2] = {kv.format == kKvQ4 ? 48u : 64u, cuuint32_t(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  return enc(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2,
             const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             f16                     ? CU_TENSOR_MAP_SWIZZLE_128B
             : kv.format == kKvI8 ? CU_TENSOR_MAP_SWIZZLE_64B
                                    : CU_TENSOR_MAP_SWIZZLE_NONE,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// q rows as [rows][hq][64] (row pitch ld), boxes of a group's heads of 128 / group rows.
bool make_q_map(CUtensorMap* m, const void* q, int hq, int64_t rows, int64_t ld, int group) {
  auto enc = get_encode();
  if (!enc) return false;
  cuuint64_t dims[3] = {64, cuuint64_t(hq), cuuint64_t(rows)};
  cuuint64_t strides[2] = {128, cuuint64_t(ld) * 2};
  cuuint32_t box[3] = {64, cuuint32_t(group), cuuint32_t(BM / group)};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(q), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

size_t chunk_parts_bytes(int num_sms) {
  return size_t(num_sms) * 2 * kRows * kRec * sizeof(float);
}
size_t chunk_join_bytes(int num_sms) { return size_t(num_sms) * sizeof(int4); }

cudaError_t launch_attn_chunk(const ChunkArgs& args, int num_sms, cudaStream_t s) {
  ChunkArgs a = args;
  const int group = a.hq / a.kv.hkv;
  CUtensorMap tq{}, tk{}, tv{};
  if (!make_q_map(&tq, a.q, a.hq, a.at.n_rows, a.ld_q, group)) return cudaErrorInvalidValue;
  const int64_t rows = a.kv.kv_rows << a.kv.shift;  // shift 0 when contiguous
  const int box = a.kv.table && (1 << a.kv.shift) < BN ? 1 << a.kv.shift : BN;
  if (rows > INT32_MAX) return cudaErrorInvalidValue;
  if (!make_map(&tk, a.kv.k, a.kv, rows, box) || !make_map(&tv, a.kv.v, a.kv, rows, box))
    return cudaErrorInvalidValue;
  struct Kernel {
    const void* fn;
    int threads, regs, smem;
  };
  auto kernel = [](auto fmt) {
    constexpr int kFmt = decltype(fmt)::value;
    using C = Conf<kFmt>;
    return Kernel{reinterpret_cast<const void*>(&attn_chunk_kernel<kFmt>), C::kThreads,
                  C::kLaunchRegs, int(sizeof(Tiles<kFmt>) + sizeof(Smem)) + 1024};
  };
  const Kernel k = a.kv.format == kKvF16  ? kernel(std::integral_constant<int, kKvF16>{})
                   : a.kv.format == kKvI8 ? kernel(std::integral_constant<int, kKvI8>{})
                                          : kernel(std::integral_constant<int, kKvQ4>{});
  static PerDeviceOnce attrs[3];
  const cudaError_t e = per_device_once(attrs[a.kv.format], [&](int&) {
    // the split of the registers needs the launch to have them all: without, a warpgroup would
    // wait for registers for good
    cudaFuncAttributes fa;
    cudaError_t r = cudaFuncGetAttributes(&fa, k.fn);
    if (r != cudaSuccess) return r;
    if (fa.numRegs != k.regs) return cudaErrorNotSupported;
    return cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem);
  });
  if (e != cudaSuccess) return e;
  void* argv[] = {&tq, &tk, &tv, &a};
  cudaError_t le = cudaLaunchKernel(k.fn, dim3(unsigned(num_sms)), dim3(unsigned(k.threads)), argv,
                                    size_t(k.smem), s);
  if (le != cudaSuccess) return le;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(num_sms), kRows / 32);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join_chunk_kernel, a);
}

}  // namespace p2p
