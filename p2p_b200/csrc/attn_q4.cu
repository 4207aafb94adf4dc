// attn_q4.cu -- attention of one token per sequence over a 4-bit KV cache (ATTN at M = 1,
// src/scripts/lfm-engine/kernels.js:268-319, optionally with QK_PREP, :216-266, in front).
//
// Mathematics.  A cached value is code * s + lo with one (s, lo) per (token, kv head), so
//     q . k_j      = s_j (q . c_j) + lo_j sum(q)
//     sum_j p_j v_j = sum_j (p_j s_j) c_j + sum_j p_j lo_j
// and only the codes c enter the tensor cores.  A 4-bit code in the low bits of an f16 is the
// subnormal c * 2^-24 (c * 2^-20 one nibble higher), which the f16 MMA multiplies exactly: a word
// of eight codes becomes four f16 pairs with one shift and four ANDs and no conversion.  The odd
// nibbles' factor 16 goes into q (divided by 16 for those dims) and into the final scale of the odd
// output dims.  A head's q enters times the power of two that puts its largest value at 2^14, taken
// out of the scores again: divided by 16 as they were, values below 2^-10 lost bits.
//     S^T[16 keys x 8 heads] = C_K[16 x 64] . Q^T[64 x 8],   O^T[64 x 8] += C_V^T[64 x 16] . P'^T
// P' = p * s goes in as a high and a low f16 in the columns that up to four query heads leave free
// (22 bits of the weight); eight heads fill the columns and P' is rounded to f16: 2^-11 of w (v - lo),
// about twice the rounding of the output where the values have no common sign.  The reference that
// weights are taken against follows the largest p * s, not the largest p, and puts it at 2^12 or more:
// a key keeps its bits down to 2^-26 of the largest weight times scale and is lost below 2^-37 of it,
// whatever the scales are.  (Against the largest p, a tail of 131071 keys of amplitude 0.03 behind a key
// 14 nats above it lost its codes: 3.5e-2 of the outputs' norm off, now 2.1e-4; it costs 2 % of the
// time.)  p, the sums of p and of p * lo, the reference and O stay in f32.
//
// Split.  All sequences' tiles, in order, form one list that is cut into equal parts, one per CTA
// (two CTAs per SM), so ragged batches balance by themselves whatever the lengths and the grid
// does not depend on them.  A CTA works on up to 8 kv heads of its tiles, one warp per head (more
// warps per head when there are fewer heads), because a page's rows are contiguous over heads:
// one bulk copy per page and pool fetches them, issued by a producer warp into a ring of stages.
// Sequences that straddle CTAs leave a record per CTA, head and query head, which a second kernel
// joins; it is launched as a programmatic dependent, so it is resident when the first one ends.  The
// order of the sums is that of the CTAs, so results repeat bit for bit, and nothing in the
// workspace outlives a call.
// What bounds it.  4 sequences of up to 131071 keys (240 MB of rows, 32 heads on 8): 59 us, 4.0 TB/s,
// 62 % of the copy rate, at 58 % of the issue slots: 470 instructions per head and 64 keys, each block
// a chain of dependent steps.  64 sequences of up to 8191 (167 MB): 47 us.  One of 1337: 9.7 us, latency.  (Three CTAs
// per SM with 72 registers were slower, and so were 32 keys a stage: 70 us.)
// Measured on the way (4 sequences, 390k keys, 8 kv heads x 4): joining by the last warp to arrive
// (a fence, an atomic and the loads of up to 16 records per level, all one after the other) took
// 8 us of a short call and 19 us of this one.
#include "common.cuh"
#include "kernels.h"
#include "kv_view.cuh"
#include "sm100.cuh"

namespace p2p {
namespace {

using sm100::fence_barrier_init;
using sm100::fence_proxy_async_smem;
using sm100::globaltimer_ns;
using sm100::mbar_arrive;
using sm100::mbar_arrive_expect_tx;
using sm100::mbar_init;
using sm100::mbar_try_wait;
using sm100::smem_u32;

constexpr int kWarps = 8;                      // compute warps; warp 8 is the producer
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kBlock = 64;                     // keys per warp and tile
constexpr int kMaxStages = 8;
constexpr int kRec = 68;                       // acc[64], max, sum, 2 pad: 17 16-byte pieces
constexpr int kJoin = 16;                      // records joined by one warp
constexpr float kNegBig = -1e30f;
// log2 of where the largest weight * scale is put when the reference is set, and from where on it is
// set again: 2^15.5 is below f16's 65504 with what add_log2_scale may be off.
constexpr float kUp = 12.f, kTop = 15.5f;
constexpr uint64_t kWaitLimitNs = 1000000000ull;

// Warps per head for a CTA of hb heads (1 .. 8); its tile is kBlock keys per such warp.
__host__ __device__ constexpr int warps_per_head(int hb) {
  return hb >= 5 ? 1 : hb >= 3 ? 2 : hb == 2 ? 4 : 8;
}
// Bytes of one token's units of hb heads, as copied and as laid out in shared memory.
__host__ __device__ constexpr int pitch_of(int hb) { return (hb * kQ4UnitBytes + 15) / 16 * 16; }
__host__ __device__ constexpr int stage_bytes(int hb) {
  return 2 * kBlock * warps_per_head(hb) * pitch_of(hb);
}

struct __align__(16) StageMeta {
  int z;        // sequence
  int key0;     // first key of the tile
  int valid;    // its keys
  int flags;    // kFirst, kLast of this CTA's part of the sequence; kBad
  long long g;  // position of the sequence's tile 0 in the list of all tiles
  int tiles;    // the sequence's tiles
  int pos;      // position of the token (its keys are 0 .. pos)
};
constexpr int kFirst = 1, kLast = 2, kBad = 4;

struct Shared {
  uint64_t full[kMaxStages], empty[kMaxStages];
  StageMeta meta[kMaxStages];
  long long wsum[kWarps];
  int z0, t0;
  volatile int abort_flag;
};

__device__ __forceinline__ bool wait_bar(Shared& s, uint64_t* bar, uint32_t parity, int32_t* err) {
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

// Untiled bulk copy: 16-byte aligned addresses, a multiple of 16 bytes.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(dst),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

constexpr uint32_t kEven = 0x000f000fu, kOdd = 0x00f000f0u;  // nibbles 0, 4 and 1, 5 of a word
// V's codes sit two bits higher, c * 2^-22 and c * 2^-18: measured, the sums of the lower nibbles were
// off by 16 times as much as those of the higher ones (a subnormal seems to be aligned by the smallest
// exponent, not by its leading bit), and two bits up leave nothing that can be seen.
constexpr uint32_t kLow = kEven << 2, kHigh = kOdd << 2;

// Query heads per lane.  Up to four heads, head t sits in lane column 2t of the fragments' eight and
// column 2t + 1 is free: it takes no score, so that a lane's softmax works on one head instead of
// two (half of them empty), and carries the low part of the weights through the P.V product.  Eight
// heads fill the columns: heads 2t and 2t + 1 are lane t's.
template <int G>
constexpr int heads_per_lane() {
  return G > 4 ? 2 : 1;
}

// A warp's query heads: B fragments of the four k-steps, and the lane's heads' sums and the factors of
// their products with the codes.
template <int H>
struct Query {
  uint32_t b[4][2];
  float sum[H], scale[H];
};

// From the G f16 rows at `q` (row stride 64): lane (gid, t) holds column gid's head, dims 8t .. 8t+7
// and 32 + 8t .. 32 + 8t + 7 in the order the code words give them.
template <int G, int H>
__device__ __forceinline__ void load_query(const __half* q, float scale_log2, Query<H>& out) {
  const int lane = threadIdx.x & 31, gid = lane >> 2, t = lane & 3;
  uint4 w[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  const int head = H == 2 ? gid : (gid & 1) ? G : gid >> 1;
  if (head < G) {
    w[0] = *reinterpret_cast<const uint4*>(q + head * 64 + 8 * t);
    w[1] = *reinterpret_cast<const uint4*>(q + head * 64 + 32 + 8 * t);
  }
  // the head's largest value, as bits; 2^14 over its power of two (1 for zeros, infinities and NaN)
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    top = __vmaxu2(top, __vmaxu2(w[i].x & 0x7fff7fffu, w[i].y & 0x7fff7fffu));
    top = __vmaxu2(top, __vmaxu2(w[i].z & 0x7fff7fffu, w[i].w & 0x7fff7fffu));
  }
  top = max(top & 0xffffu, top >> 16);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const uint32_t expo =  // of the f32
      __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(top)))) >> 23;
  const uint32_t shift = top == 0u || top >= 0x7c00u ? 127u : 141u - expo + 127u;
  const float up = __uint_as_float(shift << 23), down = __uint_as_float((254u - shift) << 23);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t d01 = w[i].x, d23 = w[i].y, d45 = w[i].z, d67 = w[i].w;
    uint32_t e[4] = {__byte_perm(d01, d45, 0x5410), __byte_perm(d01, d45, 0x7632),
                     __byte_perm(d23, d67, 0x5410), __byte_perm(d23, d67, 0x7632)};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __half2 h = *reinterpret_cast<const __half2*>(&e[k]);
      const float2 f = __half22float2(h);
      sum += f.x + f.y;
      const float by = (k & 1) ? 0.0625f * up : up;
      out.b[2 * i + (k >> 1)][k & 1] = pack_h2(f.x * by, f.y * by);
    }
  }
  sum += __shfl_xor_sync(0xffffffffu, sum, 1);
  sum += __shfl_xor_sync(0xffffffffu, sum, 2);
  sum *= scale_log2;
#pragma unroll
  for (int e = 0; e < H; ++e) {  // from a lane of column 2t + e
    out.sum[e] = __shfl_sync(0xffffffffu, sum, 8 * t + 4 * e);
    out.scale[e] = scale_log2 * 16777216.f * __shfl_sync(0xffffffffu, down, 8 * t + 4 * e);
  }
}

// kLogBias + x + log2 of the scale in a unit's parameters, from the bits of the f16: 0 to 0.09 too low
// for normal numbers, for the others as for 2^-15 (more: their rows' codes are below the output's
// rounding anyway).  The bias leaves a sum 2^-10.
constexpr float kLogBias = 8192.f + 15.f;
__device__ __forceinline__ float add_log2_scale(float x, uint32_t params) {
  // 2^23 + the bits
  const float bits = __uint_as_float(__byte_perm(params, 0x4b000000u, 0x7610));
  return fmaf(bits, 0.0009765625f, x);
}

template <int H>
struct State {
  // The reference that weights are taken against (the warp's; kUp below the largest score + log2 of
  // the value scale when it was set) and, of the lane, the sums of the weights and of weight * lo.
  float m[H], l[H], bias[H];
  // [i][c]: dim 8 gid + 2i of column 2t + c (even codes); [i][2 + c]: dim 8 gid + 2i + 1 (odd ones).
  // H = 1: the sums over the high (c = 0) and low (c = 1) parts of the weights.
  float o[4][4];
  bool fresh;  // no block yet: the reference is to be set, whatever it is
  __device__ __forceinline__ void clear() {
    fresh = true;
#pragma unroll
    for (int e = 0; e < H; ++e) m[e] = l[e] = bias[e] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  }
};

// A block of 16 NJ keys of one head: rows at ks / vs (this head's unit in the block's first key).
// Row r of the fragments is key perm(r): eight consecutive rows then read V's words of keys 2t and
// 2t + 1 from distinct banks (the row pitch is 8 banks modulo 32 for 8 heads).
// FULL: all the keys are there; else the rows behind `valid` hold whatever the stage held before and
// get neither weight nor parameters.
template <int H, bool FULL, int NJ>
__device__ __forceinline__ void attend(const unsigned char* ks, const unsigned char* vs,
                                         int pitch, int valid, const Query<H>& q, State<H>& st) {
  const int lane = threadIdx.x & 31, gid = lane >> 2, t = lane & 3;
  constexpr uint32_t kPerm = 0x57463120u;
  const int row = (kPerm >> (4 * gid)) & 7;
  float sc[2 * NJ][H];  // log2 weights of keys row, row + 8, row + 16, ...
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const uint32_t* ka = reinterpret_cast<const uint32_t*>(ks + (16 * j + row) * pitch);
    const uint32_t* kb = reinterpret_cast<const uint32_t*>(ks + (16 * j + row + 8) * pitch);
    const uint32_t a0 = ka[t], a1 = ka[t + 4], b0 = kb[t], b1 = kb[t + 4];
    const uint32_t pa = ka[8], pb = kb[8];
    float r[4] = {0.f, 0.f, 0.f, 0.f};
    mma16816(r, a0 & kEven, b0 & kEven, a0 & kOdd, b0 & kOdd, q.b[0][0], q.b[0][1]);
    mma16816(r, (a0 >> 8) & kEven, (b0 >> 8) & kEven, (a0 >> 8) & kOdd, (b0 >> 8) & kOdd,
             q.b[1][0], q.b[1][1]);
    mma16816(r, a1 & kEven, b1 & kEven, a1 & kOdd, b1 & kOdd, q.b[2][0], q.b[2][1]);
    mma16816(r, (a1 >> 8) & kEven, (b1 >> 8) & kEven, (a1 >> 8) & kOdd, (b1 >> 8) & kOdd,
             q.b[3][0], q.b[3][1]);
    float s, lo;
    q4_unpack(pa, s, lo);
#pragma unroll
    for (int e = 0; e < H; ++e)
      sc[2 * j][e] = fmaf(r[e], s * q.scale[e], fmaf(lo, q.sum[e], -st.m[e]));
    q4_unpack(pb, s, lo);
#pragma unroll
    for (int e = 0; e < H; ++e)
      sc[2 * j + 1][e] = fmaf(r[2 + e], s * q.scale[e], fmaf(lo, q.sum[e], -st.m[e]));
  }
  if (!FULL) {
#pragma unroll
    for (int k = 0; k < 2 * NJ; ++k)
      if (8 * k + row >= valid)
#pragma unroll
        for (int e = 0; e < H; ++e) sc[k][e] = -INFINITY;
  }
  uint32_t pv[2 * NJ];  // the keys' parameters of V
#pragma unroll
  for (int k = 0; k < 2 * NJ; ++k) {
    pv[k] = reinterpret_cast<const uint32_t*>(vs + (row + 8 * k) * pitch)[8];
    if (!FULL && 8 * k + row >= valid) pv[k] = 0u;
  }
  // The reference rarely has to move after the first blocks: only then are the lanes' maxima joined and
  // O rescaled.  (Scores of 2^24 and more may need it again, rounded as their differences are.)
#pragma unroll 1
  for (int pass = 0; pass < 4; ++pass) {
    float top[H];
    bool grows = st.fresh;
#pragma unroll
    for (int e = 0; e < H; ++e) {
      top[e] = add_log2_scale(sc[0][e], pv[0]);
#pragma unroll
      for (int k = 1; k < 2 * NJ; ++k) top[e] = fmaxf(top[e], add_log2_scale(sc[k][e], pv[k]));
      grows |= top[e] > kTop + kLogBias;
    }
    if (!__any_sync(0xffffffffu, grows)) break;
#pragma unroll
    for (int e = 0; e < H; ++e) {
      float most = sc[0][e];
#pragma unroll
      for (int k = 1; k < 2 * NJ; ++k) most = fmaxf(most, sc[k][e]);
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1) {
        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], o));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      }
      // a whole number away from the largest score, whose weight then is a power of two and its
      // product with the scale exact
      const float rise = most + floorf(top[e] - kLogBias - kUp - most);
      const float up = st.fresh ? rise : fmaxf(rise, 0.f);
      const float c = st.fresh ? 0.f : fast_exp2(-up);
      st.m[e] += up;
      st.l[e] *= c;
      st.bias[e] *= c;
#pragma unroll
      for (int k = 0; k < 2 * NJ; ++k) sc[k][e] -= up;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        st.o[i][e] *= c;
        st.o[i][2 + e] *= c;
        if (H == 1) {
          st.o[i][1] *= c;
          st.o[i][3] *= c;
        }
      }
    }
    st.fresh = false;
  }
  // A block's products are summed apart and then added: the MMA truncates what it adds to its
  // accumulators, and codes are never negative, so over thousands of keys the losses of a running sum
  // would all go one way (4 x 131071 keys: 6.5e-4 of the outputs' norm from
  // the exact ones; summed apart 2.1e-4, which is the rounding to f16).
  float o[4][4] = {};
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    // weights of keys row and row + 8 of this half, scaled by the keys' value scales: columns 2t
    // and 2t + 1 of the fragment
    uint32_t w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float s, lo, ps[2];
      q4_unpack(pv[2 * j + k], s, lo);
#pragma unroll
      for (int e = 0; e < H; ++e) {
        const float p = fast_exp2(sc[2 * j + k][e]);
        st.l[e] += p;
        st.bias[e] = fmaf(p, lo, st.bias[e]);
        ps[e] = p * s;
      }
      if (H == 1) {  // high and low part: 22 bits of the weight
        const float hi = __half2float(__float2half_rn(ps[0]));
        ps[1] = ps[0] - hi;
      }
      w[k] = pack_h2(ps[0], ps[1]);
    }
    const uint32_t b0 = movmatrix_trans(w[0]), b1 = movmatrix_trans(w[1]);
    const unsigned char* v0 = vs + (16 * j + ((kPerm >> (8 * t)) & 7)) * pitch + 4 * gid;
    const unsigned char* v1 = vs + (16 * j + ((kPerm >> (8 * t + 4)) & 7)) * pitch + 4 * gid;
    const uint32_t w0 = *reinterpret_cast<const uint32_t*>(v0);
    const uint32_t w1 = *reinterpret_cast<const uint32_t*>(v1);
    const uint32_t w2 = *reinterpret_cast<const uint32_t*>(v0 + 8 * pitch);
    const uint32_t w3 = *reinterpret_cast<const uint32_t*>(v1 + 8 * pitch);
    // pairs of keys: codes 0..3 of both words, then codes 4..7
    const uint32_t x = __byte_perm(w0, w1, 0x5410), y = __byte_perm(w0, w1, 0x7632);
    const uint32_t x2 = __byte_perm(w2, w3, 0x5410), y2 = __byte_perm(w2, w3, 0x7632);
    mma16816(o[0], (x << 2) & kLow, (x << 2) & kHigh, (x2 << 2) & kLow, (x2 << 2) & kHigh, b0, b1);
    mma16816(o[1], (x >> 6) & kLow, (x >> 6) & kHigh, (x2 >> 6) & kLow, (x2 >> 6) & kHigh, b0, b1);
    mma16816(o[2], (y << 2) & kLow, (y << 2) & kHigh, (y2 << 2) & kLow, (y2 << 2) & kHigh, b0, b1);
    mma16816(o[3], (y >> 6) & kLow, (y >> 6) & kHigh, (y2 >> 6) & kLow, (y2 >> 6) & kHigh, b0, b1);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) st.o[i][k] += o[i][k];
}

// A warp's part of one head's G query heads as a record [G][acc[64] | max | sum]: from the
// fragments (acc[e][i]: dim 8 gid + i of the lane's head e) ...
template <int G, int H>
__device__ __forceinline__ void store_fragments(float* rec, const float (&acc)[H][8],
                                                const float (&m)[H], const float (&l)[H]) {
  const int lane = threadIdx.x & 31, gid = lane >> 2, t = lane & 3;
#pragma unroll
  for (int e = 0; e < H; ++e) {
    const int g = H * t + e;
    if (g >= G) continue;
    float* r = rec + g * kRec;
    *reinterpret_cast<float4*>(r + 8 * gid) =
        make_float4(acc[e][0], acc[e][1], acc[e][2], acc[e][3]);
    *reinterpret_cast<float4*>(r + 8 * gid + 4) =
        make_float4(acc[e][4], acc[e][5], acc[e][6], acc[e][7]);
    if (gid == 0) *reinterpret_cast<float2*>(r + 64) = make_float2(m[e], l[e]);
  }
}

// ... or joined from several: piece lane + 32 k of the G x 16 16-byte pieces, so that a record is
// one or a few coalesced loads of the warp.  Piece k belongs to head 2k + lane / 16.
template <int G>
struct Joined {
  static constexpr int kPieces = (G + 1) / 2;
  float4 acc[kPieces];
  float m[kPieces], l[kPieces];  // l < 0: some page of the sequence was refused

  __device__ __forceinline__ static bool has(int k) { return G > 1 || (threadIdx.x & 31) < 16; }
  __device__ __forceinline__ static int head(int k) {
    return G > 1 ? 2 * k + ((threadIdx.x & 31) >> 4) : 0;
  }

  __device__ __forceinline__ void none() {
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      m[k] = kNegBig;
      l[k] = 0.f;
    }
  }
  __device__ __forceinline__ void add(const Joined& x) {
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const float mx = fmaxf(m[k], x.m[k]);
      const float c = fast_exp2(m[k] - mx), d = fast_exp2(x.m[k] - mx);
      l[k] = l[k] < 0.f || x.l[k] < 0.f ? -1.f : fmaf(l[k], c, x.l[k] * d);
      m[k] = mx;
      acc[k].x = fmaf(acc[k].x, c, x.acc[k].x * d);
      acc[k].y = fmaf(acc[k].y, c, x.acc[k].y * d);
      acc[k].z = fmaf(acc[k].z, c, x.acc[k].z * d);
      acc[k].w = fmaf(acc[k].w, c, x.acc[k].w * d);
    }
  }
  // The n <= kJoin records rec(i), in order.  Lane i (and i + 16) first takes record i's maximum
  // and sum, so that all of them are one load; then the accumulators, several records in flight.
  template <bool GLOBAL, class Rec>
  __device__ __forceinline__ void join(int n, Rec rec) {
    const int lane = threadIdx.x & 31;
    float c[kPieces];
    const float* mine = rec(min(lane & 15, n - 1));
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      float2 ml;
      if (GLOBAL) ml = __ldcg(reinterpret_cast<const float2*>(mine + head(k) * kRec + 64));
      else ml = *reinterpret_cast<const float2*>(mine + head(k) * kRec + 64);
      if ((lane & 15) >= n) ml = make_float2(kNegBig, 0.f);
      m[k] = ml.x;
      l[k] = ml.y;
    }
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const uint32_t refused = __ballot_sync(0xffffffffu, l[k] < 0.f);
      float mx = m[k];
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      c[k] = fast_exp2(m[k] - mx);
      float sum = l[k] * c[k];
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      m[k] = mx;
      l[k] = ((refused >> (lane & 16)) & 0xffffu) ? -1.f : sum;
      acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    constexpr int kBatch = kPieces > 2 ? 4 : 8;
    for (int i0 = 0; i0 < n; i0 += kBatch) {
      float4 x[kBatch][kPieces];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float* r = rec(min(i0 + i, n - 1));
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
          const float4* p = reinterpret_cast<const float4*>(r + head(k) * kRec) + (lane & 15);
          if (GLOBAL) x[i][k] = __ldcg(p);
          else x[i][k] = *p;
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
          // 0 behind the last record: lanes n .. 15 hold exp2(-1e30 - max)
          const float w = __shfl_sync(0xffffffffu, c[k], min(i0 + i, 15) | (lane & 16));
          if (i0 + i < n) {
            acc[k].x = fmaf(x[i][k].x, w, acc[k].x);
            acc[k].y = fmaf(x[i][k].y, w, acc[k].y);
            acc[k].z = fmaf(x[i][k].z, w, acc[k].z);
            acc[k].w = fmaf(x[i][k].w, w, acc[k].w);
          }
        }
    }
  }
  __device__ __forceinline__ void store(float* rec) const {
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      if (!has(k)) continue;
      float* r = rec + head(k) * kRec;
      reinterpret_cast<float4*>(r)[threadIdx.x & 15] = acc[k];
      if ((threadIdx.x & 15) == 0) *reinterpret_cast<float2*>(r + 64) = make_float2(m[k], l[k]);
    }
  }
  __device__ __forceinline__ void write(__half* out) const {  // [G][64]
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      if (!has(k) || l[k] < 0.f) continue;
      const float inv = __fdiv_rn(1.f, l[k]);
      reinterpret_cast<uint2*>(out + head(k) * 64)[threadIdx.x & 15] =
          make_uint2(pack_h2(acc[k].x * inv, acc[k].y * inv),
                     pack_h2(acc[k].z * inv, acc[k].w * inv));
    }
  }
};

// The tiles of a CTA's part, in order, sequence by sequence.  The next sequence's length and offset
// are loaded while this one's tiles go by.
struct Walk {
  const KvView& kv;
  const ChunkIndex& at;
  int tile, z, t, tiles, off, next_past, next_off;
  SeqSpan sp;
  __device__ __forceinline__ Walk(const KvView& k, const ChunkIndex& x, int tile_, int z0, int t0)
      : kv(k), at(x), tile(tile_), z(z0), t(t0) {
    fetch(z0);
    take();
  }
  __device__ __forceinline__ void fetch(int i) {
    next_past = i < at.nseq ? at.past[i] : -1;
    next_off = kv.table == nullptr && i < at.nseq ? kv.offsets[i] : 0;
  }
  __device__ __forceinline__ void take() {
    sp.past = next_past;
    off = next_off;
    sp.ok = one_token_fits(kv, at, sp.past, off);
    tiles = (sp.past + tile) / tile;  // of past + 1 keys
    fetch(z + 1);
  }
  // Moves on to the next sequence that has tiles when this one's are done.
  __device__ __forceinline__ void settle() {
    if (t < tiles) return;
    do {
      ++z;
      take();
    } while (!sp.ok && z < at.nseq);
    t = 0;
  }
};

// The record of head h of CTA b (of `ctas` per group of heads): slot 0 its first sequence, 1 its
// last.
__device__ __forceinline__ int64_t record_of(int grp, int ctas, int b, int slot, int h) {
  return ((int64_t(grp) * ctas + b) * 2 + slot) * 8 + h;
}

// HB: the kv heads of every group when that number is 8, 4, 2 or 1 (row pitches are then constants
// in the addresses), or 0.
template <int G, bool FUSED, int HB>
__global__ void __launch_bounds__(kThreads, 2)
    attn_decode_q4_kernel(const __grid_constant__ DecodeQ4Args a) {
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ Shared s;
  __shared__ __align__(16) __half q_s[FUSED ? kWarps : 1][FUSED ? G : 1][64];
  __shared__ __align__(16) __half new_s[FUSED ? kWarps : 1][2][64];
  __shared__ uint32_t unit_s[FUSED ? kWarps : 1][2][9];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int grp = blockIdx.y;
  const int hb = HB ? HB : min(8, a.kv.hkv - 8 * grp), wph = warps_per_head(hb);
  const int tile = kBlock * wph, pitch = pitch_of(hb), sbytes = 2 * tile * pitch;
  const int n_groups = gridDim.y;

  // ---- the CTA's part of the list of tiles
  const int per = (a.at.nseq + kWarps * 32 - 1) / (kWarps * 32);
  long long mine = 0, upto = 0;
  if (tid == 0) {
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], kWarps);
    }
    s.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp < kWarps) {
    for (int z = tid * per; z < min((tid + 1) * per, a.at.nseq); ++z) {
      const SeqSpan sp = seq_span(a.kv, a.at, z);
      if (sp.ok) mine += (sp.past + tile) / tile;  // tiles of past + 1 keys
      else if (blockIdx.x == 0 && grp == 0) atomicOr(a.err, kErrPosBeyondCache);
    }
    upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) s.wsum[warp] = upto;
  }
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) upto += total;
    total += s.wsum[w];
  }
  const int parts = int(min(static_cast<long long>(gridDim.x), total));
  const int b = blockIdx.x;
  launch_dependents();  // the joining kernel may take the slots that become free
  if (tid == 0) a.joins[grp * gridDim.x + b] = make_int4(-1, 0, 0, 0);
  if (b >= parts) return;
  const long long lo = total * b / parts;
  const int n_tiles = int(total * (b + 1) / parts - lo);
  if (warp < kWarps && lo < upto && lo >= upto - mine) {
    long long at = upto - mine;
    for (int z = tid * per;; ++z) {
      const SeqSpan sp = seq_span(a.kv, a.at, z);
      const int tz = sp.ok ? (sp.past + tile) / tile : 0;
      if (lo < at + tz) {
        s.z0 = z;
        s.t0 = int(lo - at);
        break;
      }
      at += tz;
    }
  }
  __syncthreads();

  if (warp == kWarps) {
    // ------------------------------------------------------------------ producer
    Walk w(a.kv, a.at, tile, s.z0, s.t0);
    // keys of one contiguous run: the cache's rows are whole tokens, so a run can span keys only
    // when one group of heads is the whole row
    const bool paged = a.kv.table != nullptr;
    const int shift = a.kv.shift;
    const int run = n_groups > 1 ? 1 : paged ? min(1 << shift, tile) : tile;
    // The block table's entries pass through a window of 32 in the lanes, with the next 32 on their
    // way: a load per tile would put its latency (more than a tile takes) in front of every copy.
    // A tile covers 1 to 32 pages (a power of two), or part of one, so it never straddles two windows.
    int page0 = 0;
    int32_t pages = 0, next_pages = 0;
    auto table_at = [&](int z, int p) {
      return p < a.kv.max_blocks ? a.kv.table[int64_t(z) * a.kv.max_blocks + p] : -1;
    };
    int issued = 0, st = 0;
    uint32_t round = 0;  // parity of the stages' current use
    for (int i = 0; i < n_tiles; ++i, ++w.t) {
      w.settle();
      const int z = w.z, key0 = w.t * tile, len = w.sp.past + 1, valid = min(tile, len - key0);
      const int n_copy = FUSED && key0 + valid == len ? valid - 1 : valid;
      if (paged) {
        const int p = key0 >> shift;
        if (i == 0 || w.t == 0) {
          page0 = p;
          pages = table_at(z, p + lane);
          next_pages = table_at(z, p + 32 + lane);
        } else if (p >= page0 + 32) {
          page0 += 32;
          pages = next_pages;
          next_pages = table_at(z, page0 + 32 + lane);
        }
      }
      // cache row of the tile's key k, -1 when its page is outside the pool (whole warps call it)
      auto row_at = [&](int k) -> int64_t {
        const int pos = key0 + k;
        if (!paged) return int64_t(w.off) + pos;
        const int32_t pg = __shfl_sync(0xffffffffu, pages, (pos >> shift) - page0);
        if (pg < 0 || int64_t(pg) >= a.kv.kv_rows) return -1;
        return (int64_t(pg) << shift) | (pos & ((1 << shift) - 1));
      };
      bool bad = false;
      for (int k = 0; k < valid; k += 32 * run) {
        const int mine = k + lane * run;
        bad |= row_at(min(mine, valid - 1)) < 0;
      }
      bad = __any_sync(0xffffffffu, bad);
      if (i >= a.stages) {
        bool ok = true;
        if (lane == 0) ok = wait_bar(s, &s.empty[st], round ^ 1, a.err);
        if (!__shfl_sync(0xffffffffu, ok ? 1 : 0, 0)) break;
      }
      if (lane == 0) {
        if (bad) atomicOr(a.err, kErrPosBeyondCache);
        StageMeta& m = s.meta[st];
        m.z = z;
        m.key0 = key0;
        m.valid = valid;
        m.flags = (i == 0 || w.t == 0 ? kFirst : 0) |
                  (i == n_tiles - 1 || w.t == w.tiles - 1 ? kLast : 0) | (bad ? kBad : 0);
        m.g = lo + i - w.t;
        m.tiles = w.tiles;
        m.pos = w.sp.past;
        mbar_arrive_expect_tx(&s.full[st],
                              uint32_t(bad ? 0 : 2 * n_copy * pitch) +
                                  uint32_t(i == 0 ? a.wait_deficit : 0));
      }
      __syncwarp();
      if (!bad) {
        const uint32_t dst = smem_u32(ring) + uint32_t(st * sbytes);
        const int runs = (n_copy + run - 1) / run;
        for (int k0 = 0; k0 < 2 * runs; k0 += 32) {
          const int k = k0 + lane, pool = k >= runs, r = k - pool * runs;
          const int64_t row = row_at(min(r * run, valid - 1));
          if (k < 2 * runs)
            bulk_load(dst + uint32_t((pool * tile + r * run) * pitch),
                      (pool ? a.kv.v : a.kv.k) + row * a.kv.row_bytes + grp * 8 * kQ4UnitBytes,
                      uint32_t(min(run, n_copy - r * run) * pitch), &s.full[st]);
        }
      }
      issued = i + 1;
      if (++st == a.stages) {
        st = 0;
        round ^= 1;
      }
    }
    if (s.abort_flag) {  // let the copies already in flight land before the CTA exits
      for (int i = max(0, issued - a.stages); i < issued; ++i) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&s.full[i % a.stages], (i / a.stages) & 1) &&
               globaltimer_ns() - t0 < kWaitLimitNs) {
        }
      }
    }
    return;
  }

  // -------------------------------------------------------------------- compute warps
  const int h = warp % hb, sub = warp / hb;
  const bool active = sub < wph;
  const int kh = grp * 8 + h;
  constexpr int H = heads_per_lane<G>();
  Query<H> q;
  State<H> state;
  bool bad = false;
  int segs = 0;  // parts of sequences ended
  float* merge = reinterpret_cast<float*>(ring + a.stages * a.stage_bytes);  // [warp][G][kRec]
  auto out_of = [&](int z) { return a.out + int64_t(z) * a.ld_o + kh * G * 64; };
  auto whole = [&](long long g0, int tiles) { return lo <= g0 && lo + n_tiles >= g0 + tiles; };
  // Ends this CTA's part of sequence z (whose `tiles` tiles begin at g0 of the list): the warps of
  // a head meet, and the output is written, or a record when other CTAs have parts of it too.
  auto end_part = [&](const float (&acc)[H][8], const float (&m)[H], const float (&l)[H], int z,
                      long long g0, int tiles, bool seg_first) {
    float* own = a.parts + record_of(grp, gridDim.x, b, seg_first ? 0 : 1, h) * (G * kRec);
    if (tid == 0 && lo <= g0 && !whole(g0, tiles)) {  // it begins here: what there is to join
      const int last = int(((g0 + tiles) * parts - 1) / total);  // the CTA of its last tile
      a.joins[grp * gridDim.x + b] = make_int4(z, seg_first ? 0 : 1, last - b + 1, 0);
    }
    if (wph > 1) {
      if (active) store_fragments<G>(merge + warp * G * kRec, acc, m, l);
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (sub == 0) {
        Joined<G> j;
        j.template join<false>(wph, [&](int k) { return merge + (k * hb + h) * G * kRec; });
        if (whole(g0, tiles)) j.write(out_of(z));
        else j.store(own);
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
    } else if (active) {
      if (!whole(g0, tiles)) {
        store_fragments<G>(own, acc, m, l);
      } else {
        const int gid = lane >> 2, t = lane & 3;
#pragma unroll
        for (int e = 0; e < H; ++e) {
          if (H * t + e >= G || l[e] < 0.f) continue;
          const float inv = __fdiv_rn(1.f, l[e]);
          *reinterpret_cast<uint4*>(out_of(z) + (H * t + e) * 64 + 8 * gid) =
              make_uint4(pack_h2(acc[e][0] * inv, acc[e][1] * inv),
                         pack_h2(acc[e][2] * inv, acc[e][3] * inv),
                         pack_h2(acc[e][4] * inv, acc[e][5] * inv),
                         pack_h2(acc[e][6] * inv, acc[e][7] * inv));
        }
      }
    }
  };
  int i = 0, st = 0;
  uint32_t round = 0;
  int z = s.z0, tiles = 0;  // the sequence at hand
  long long g0 = 0;
  state.clear();
  q = Query<H>{};
  for (; i < n_tiles; ++i) {
    const bool ok = wait_bar(s, &s.full[st], round, a.err);
    if (!__all_sync(0xffffffffu, ok)) break;
    const StageMeta& m = s.meta[st];
    const int4 head = *reinterpret_cast<const int4*>(&m);  // z, key0, valid, flags
    const int flags = head.w;
    int pos = 0;
    if (flags & (kFirst | kLast)) {
      z = head.x;
      pos = m.pos;
      tiles = m.tiles;
      g0 = m.g;
    }
    unsigned char* ks = ring + st * sbytes + sub * (tile / wph) * pitch + h * kQ4UnitBytes;
    unsigned char* vs = ks + tile * pitch;
    // the sequence's last tile ends this part
    const bool has_new = FUSED && (flags & kLast) && head.y + head.z == pos + 1;
    if (flags & kFirst) {
      if (active) {
        const __half* row = a.q + int64_t(z) * a.ld_q;
        if (FUSED) {
          const float cs = to_f32(a.rope[int64_t(pos) * 64 + lane]);
          const float sn = to_f32(a.rope[int64_t(pos) * 64 + 32 + lane]);
          const __half* src = row + kh * G * 64;
          float x[G][2];
#pragma unroll
          for (int g = 0; g < G; ++g) {
            x[g][0] = to_f32(src[g * 64 + lane]);
            x[g][1] = to_f32(src[g * 64 + 32 + lane]);
          }
          const bool nw = a.norm_w != nullptr;
          const float w0 = nw ? to_f32(a.norm_w[lane]) : 0.f;
          const float w1 = nw ? to_f32(a.norm_w[32 + lane]) : 0.f;
          __syncwarp();  // q_s of the sequence before has been read
#pragma unroll
          for (int g = 0; g < G; ++g) {
            float r0, r1;
            norm_rope_vals<__half>(x[g][0], x[g][1], w0, w1, nw, a.eps, cs, sn, r0, r1);
            q_s[warp][g][lane] = __float2half_rn(r0);
            q_s[warp][g][32 + lane] = __float2half_rn(r1);
          }
          __syncwarp();
          load_query<G, H>(&q_s[warp][0][0], a.scale_log2, q);
        } else {
          load_query<G, H>(row + kh * G * 64, a.scale_log2, q);
        }
      }
    }
    if (flags & kBad) bad = true;
    int valid = head.z - sub * (tile / wph);
    if (!active || bad) valid = 0;
    if (FUSED && has_new) {
      const int at = valid - 1;  // the new token's row, if it is among this warp's
      if (at >= 0 && at < tile / wph) {
        // the new token's unit of this head: normed, rotated, quantised, into the cache and over
        // the stage's row (which the copy left out)
        const __half* row = a.q + int64_t(z) * a.ld_q;
        const float cs = to_f32(a.rope[int64_t(pos) * 64 + lane]);
        const float sn = to_f32(a.rope[int64_t(pos) * 64 + 32 + lane]);
        const __half* kn = row + (a.hq + kh) * 64;
        const __half* vn = row + (a.hq + a.kv.hkv + kh) * 64;
        float r0, r1;
        norm_rope_head<__half>(to_f32(kn[lane]), to_f32(kn[32 + lane]),
                               a.norm_w ? a.norm_w + 64 : nullptr, a.norm_w != nullptr, a.eps, cs,
                               sn, r0, r1);
        __syncwarp();
        new_s[warp][0][lane] = __float2half_rn(r0);
        new_s[warp][0][32 + lane] = __float2half_rn(r1);
        new_s[warp][1][lane] = vn[lane];
        new_s[warp][1][32 + lane] = vn[32 + lane];
        __syncwarp();
        float x[8];  // lanes 0-7: k's unit, 8-15: v's (the others repeat them)
        const int sl = lane & 7, kv = (lane >> 3) & 1;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[k] = to_f32(new_s[warp][kv][4 * sl + k]);
          x[4 + k] = to_f32(new_s[warp][kv][32 + 4 * sl + k]);
        }
        q4_store_unit(x, unit_s[warp][kv], lane < 16);
        __syncwarp();
        if (lane < 18) {
          const int pool = lane / 9, w = lane % 9;
          const uint32_t v = unit_s[warp][pool][w];
          const int64_t cached = kv_row(a.kv, z, pos);
          reinterpret_cast<uint32_t*>((pool ? a.kv.v : a.kv.k) + cached * a.kv.row_bytes +
                                      kh * kQ4UnitBytes)[w] = v;
          reinterpret_cast<uint32_t*>((pool ? vs : ks) + at * pitch)[w] = v;
        }
        fence_proxy_async_smem();  // a later copy into this stage comes after these writes
        __syncwarp();
      }
    }
    if (valid >= kBlock) {
      attend<H, true, 4>(ks, vs, pitch, kBlock, q, state);
    } else {  // the sequence's last keys, in two halves
      for (int k = 0; k < 2 && valid > 0; ++k, valid -= kBlock / 2) {
        attend<H, false, 2>(ks, vs, pitch, valid, q, state);
        ks += kBlock / 2 * pitch;
        vs += kBlock / 2 * pitch;
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.empty[st]);
    if (++st == a.stages) {
      st = 0;
      round ^= 1;
    }
    if (!(flags & kLast)) continue;

    // ---- this CTA's part of the sequence is done
    float acc[H][8], mx[H], sum[H];
#pragma unroll
    for (int e = 0; e < H; ++e) {
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1) {
        state.l[e] += __shfl_xor_sync(0xffffffffu, state.l[e], o);
        state.bias[e] += __shfl_xor_sync(0xffffffffu, state.bias[e], o);
      }
      mx[e] = state.fresh ? kNegBig : state.m[e];
      sum[e] = bad ? -1.f : state.l[e];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float even = H == 2 ? state.o[k][e] : state.o[k][0] + state.o[k][1];
        const float odd = H == 2 ? state.o[k][2 + e] : state.o[k][2] + state.o[k][3];
        acc[e][2 * k] = fmaf(even, 4194304.f, state.bias[e]);     // 2^22
        acc[e][2 * k + 1] = fmaf(odd, 262144.f, state.bias[e]);   // 2^18
      }
    }
    end_part(acc, mx, sum, z, g0, tiles, segs == 0);
    ++segs;
    state.clear();
    q = Query<H>{};
    bad = false;
  }
  if (i < n_tiles) {
    // A wait ran out: the parts that are left end as bad ones, so that no other warp waits in vain and
    // the joining kernel writes none of them.
    Walk w(a.kv, a.at, tile, s.z0, s.t0);
    int done = segs;
    for (int k = 0; k < n_tiles; ++k, ++w.t) {
      w.settle();
      if (!(k == n_tiles - 1 || w.t == w.tiles - 1) || done-- > 0) continue;
      float acc[H][8] = {}, mx[H], sum[H];
#pragma unroll
      for (int e = 0; e < H; ++e) mx[e] = kNegBig, sum[e] = -1.f;
      z = w.z;
      g0 = lo + k - w.t;
      tiles = w.tiles;
      end_part(acc, mx, sum, z, g0, tiles, segs == 0);
      ++segs;
    }
  }
}

// CTA (c, h): joins head h of the sequences that began in CTAs kJoinWarps c .. of the first kernel
// and went on in others.  Up to kJoin records are one warp's; more are spread over the warps, which
// meet in shared memory.
constexpr int kJoinWarps = 8;
template <int G>
__global__ void __launch_bounds__(kJoinWarps * 32)
    join_q4_kernel(const float* parts, const int4* joins, __half* out, int64_t ld_o, int hkv,
                   int ctas) {
  __shared__ __align__(16) float meet[kJoinWarps][G * kRec];
  __shared__ int4 many[kJoinWarps];
  const int warp = threadIdx.x >> 5, b0 = blockIdx.x * kJoinWarps, kh = blockIdx.y;
  const int grp = kh >> 3, h = kh & 7;
  grid_dependency_wait();
  // sequence (-1: none), first slot, records
  int4 d = make_int4(-1, 0, 0, 0);
  if (b0 + warp < ctas) d = joins[grp * ctas + b0 + warp];
  if ((threadIdx.x & 31) == 0) many[warp] = d.x >= 0 && d.z > kJoin ? d : make_int4(-1, 0, 0, 0);
  auto rec = [&](int b, int slot, int i) {
    return parts + record_of(grp, ctas, b + i, i == 0 ? slot : 0, h) * (G * kRec);
  };
  Joined<G> j;
  if (d.x >= 0 && d.z <= kJoin) {
    j.template join<true>(d.z, [&](int k) { return rec(b0 + warp, d.y, k); });
    j.write(out + int64_t(d.x) * ld_o + kh * G * 64);
  }
  __syncthreads();
  for (int w = 0; w < kJoinWarps; ++w) {
    d = many[w];
    if (d.x < 0) continue;
    j.none();
    for (int i0 = warp; i0 < d.z; i0 += kJoinWarps * kJoin) {
      Joined<G> x;
      x.template join<true>(min(kJoin, (d.z - i0 + kJoinWarps - 1) / kJoinWarps),
                            [&](int k) { return rec(b0 + w, d.y, i0 + k * kJoinWarps); });
      j.add(x);
    }
    j.store(meet[warp]);
    __syncthreads();
    if (warp == 0) {
      j.template join<false>(kJoinWarps, [&](int k) { return meet[k]; });
      j.write(out + int64_t(d.x) * ld_o + kh * G * 64);
    }
    __syncthreads();
  }
}

struct Pick {
  const void* fn;
  int id;  // of 4 groups x 2 x 5 head counts
};
template <int G, int HB>
const void* pick(bool fused) {
  return fused ? reinterpret_cast<const void*>(&attn_decode_q4_kernel<G, true, HB>)
               : reinterpret_cast<const void*>(&attn_decode_q4_kernel<G, false, HB>);
}
template <int G>
Pick pick(bool fused, int hb) {
  const int id = fused ? 5 : 0;
  switch (hb) {
    case 8: return {pick<G, 8>(fused), id};
    case 4: return {pick<G, 4>(fused), id + 1};
    case 2: return {pick<G, 2>(fused), id + 2};
    case 1: return {pick<G, 1>(fused), id + 3};
    default: return {pick<G, 0>(fused), id + 4};
  }
}
Pick pick(int group, bool fused, int hkv) {
  const int hb = hkv % 8 == 0 ? 8 : hkv < 8 ? hkv : 0;
  Pick p{nullptr, 0};
  switch (group) {
    case 1: p = pick<1>(fused, hb); break;
    case 2: p = pick<2>(fused, hb); p.id += 10; break;
    case 4: p = pick<4>(fused, hb); p.id += 20; break;
    case 8: p = pick<8>(fused, hb); p.id += 30; break;
  }
  return p;
}

constexpr int kSmemBytes = 113 * 1024;  // of a CTA, static ones included: two CTAs per SM

}  // namespace

int decode_q4_ctas(int num_sms, int hkv) {
  const int groups = (hkv + 7) / 8;
  return groups > 2 * num_sms ? 0 : 2 * num_sms / groups;
}

size_t decode_q4_parts_bytes(int num_sms) {
  return size_t(2 * num_sms) * 2 * 8 * 8 * kRec * sizeof(float);
}
size_t decode_q4_join_bytes(int num_sms) { return size_t(2 * num_sms) * sizeof(int4); }

cudaError_t launch_decode_q4(const DecodeQ4Args& args, int num_sms, cudaStream_t s) {
  DecodeQ4Args a = args;
  const int group = a.hq / a.kv.hkv, groups = (a.kv.hkv + 7) / 8;
  const Pick k = pick(group, a.fused != 0, a.kv.hkv);
  const void* fn = k.fn;
  const int ctas = decode_q4_ctas(num_sms, a.kv.hkv);
  if (!fn || ctas < 1) return cudaErrorInvalidValue;
  // the groups' stages: 8 heads each, the last one the rest
  const int rest = a.kv.hkv - 8 * (groups - 1);
  a.stage_bytes = stage_bytes(rest);
  if (groups > 1 && a.stage_bytes < stage_bytes(8)) a.stage_bytes = stage_bytes(8);
  const int merge = warps_per_head(rest) > 1 ? kWarps * group * kRec * 4 : 0;
  static PerDeviceOnce attrs[40];
  int fixed = 0;  // the kernel's static shared memory
  const cudaError_t e = per_device_once(attrs[k.id], [&](int& value) {
    cudaFuncAttributes fa;
    cudaError_t r = cudaFuncGetAttributes(&fa, fn);
    if (r != cudaSuccess) return r;
    value = int(fa.sharedSizeBytes);
    return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kSmemBytes - value);
  }, &fixed);
  if (e != cudaSuccess) return e;
  a.stages = (kSmemBytes - fixed - merge) / a.stage_bytes;
  if (a.stages < 1) return cudaErrorInvalidValue;  // (1 for one kv head of 8 query heads)
  if (a.stages > kMaxStages) a.stages = kMaxStages;
  const size_t smem = size_t(a.stages) * a.stage_bytes + merge;
  void* argv[] = {&a};
  cudaError_t le = cudaLaunchKernel(fn, dim3(unsigned(ctas), unsigned(groups)), dim3(kThreads),
                                    argv, smem, s);
  if (le != cudaSuccess) return le;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned((ctas + kJoinWarps - 1) / kJoinWarps), unsigned(a.kv.hkv));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  const float* pp = a.parts;
  const int4* pj = a.joins;
  auto join = [&](auto kernel) {
    return cudaLaunchKernelEx(&cfg, kernel, pp, pj, a.out, a.ld_o, a.kv.hkv, ctas);
  };
  return group == 1   ? join(&join_q4_kernel<1>)
         : group == 2 ? join(&join_q4_kernel<2>)
         : group == 4 ? join(&join_q4_kernel<4>)
                      : join(&join_q4_kernel<8>);
}

}  // namespace p2p
