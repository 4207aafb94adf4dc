// serve_api.cu -- the C entry points of the batched serving operators: caches of any layout
// (append, read back, 4-bit conversion, prompt-chunk attention) and the tokens of a batch of
// logits.  Host-side checks only; the kernels check what lives in device memory.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>

// The library is built with -fvisibility=hidden; only the declared C ABI is exported.
#pragma GCC visibility push(default)
#include "../../include/p2p_attn.h"
#pragma GCC visibility pop
#include "host_internal.h"
#include "kernels.h"
#include "rows.h"

static_assert(P2P_MAX_VOCAB == p2p::kMaxVocab, "vocabulary limit");
static_assert(P2P_KV_F16 == int(p2p::kKvF16) && P2P_KV_I8 == int(p2p::kKvI8) &&
                  P2P_KV_Q4 == int(p2p::kKvQ4),
              "cache formats");

namespace {

p2p_status fail(p2p_ctx* ctx, p2p_status s, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return p2p::ctx_fail(ctx, s, buf);
}

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Makes the context's device current for a call.
struct OnDevice {
  int prev = -1;
  bool ok = true;
  explicit OnDevice(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) ok = cudaSetDevice(dev) == cudaSuccess;
    else prev = -1;
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

p2p_status launched(p2p_ctx* ctx, cudaError_t e, const char* who) {
  if (e == cudaSuccess) return P2P_OK;
  return fail(ctx, P2P_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}

}  // namespace

namespace p2p {

p2p_status make_kv_view(p2p_ctx* ctx, const p2p_kv_layout* lay, int32_t hkv, const void* k,
                        const void* v, int64_t kv_rows, const int32_t* offsets, int32_t nseq,
                        const char* who, KvView* out) {
  if (!lay) return fail(ctx, P2P_ERR_INVALID_ARG, "%s: layout is NULL", who);
  if (lay->format != P2P_KV_F16 && lay->format != P2P_KV_I8 && lay->format != P2P_KV_Q4)
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: format %d", who, lay->format);
  if (!k || !v || kv_rows <= 0)
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: NULL cache or kv_rows %lld", who,
                (long long)kv_rows);
  if (!aligned(k, 16) || !aligned(v, 16))
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: cache buffers must be 16-byte aligned", who);
  if (nseq < 0 || nseq > 65535) return fail(ctx, P2P_ERR_INVALID_ARG, "%s: nseq %d", who, nseq);
  KvView c{};
  if (lay->block_size != 0) {
    const int bs = lay->block_size;
    if (bs < 16 || bs > 4096 || (bs & (bs - 1)) || (!lay->block_table && nseq > 0) ||
        lay->max_blocks <= 0)
      return fail(ctx, P2P_ERR_INVALID_ARG,
                  "%s: block_size %d (a power of two in 16..4096), block table %p, max_blocks %d",
                  who, bs, (const void*)lay->block_table, lay->max_blocks);
    c.table = lay->block_table;
    c.max_blocks = lay->max_blocks;
    while ((1 << c.shift) < bs) ++c.shift;
  } else if (!offsets && nseq > 0) {
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: contiguous caches need offsets", who);
  }
  if (lay->format == P2P_KV_I8) {
    const int chan = hkv * 64;
    if (!lay->k_scale || !lay->v_scale || (lay->scale_count != 1 && lay->scale_count != chan))
      return fail(ctx, P2P_ERR_INVALID_ARG,
                  "%s: int8 caches need k/v scales, 1 or %d of them (got %d)", who, chan,
                  lay->scale_count);
    if (!aligned(lay->k_scale, 4) || !aligned(lay->v_scale, 4))
      return fail(ctx, P2P_ERR_INVALID_ARG, "%s: scales not aligned to their type", who);
    c.k_scale = lay->k_scale;
    c.v_scale = lay->v_scale;
    c.per_channel = lay->scale_count > 1 ? 1 : 0;
  }
  c.k = static_cast<unsigned char*>(const_cast<void*>(k));
  c.v = static_cast<unsigned char*>(const_cast<void*>(v));
  c.kv_rows = kv_rows;
  c.row_bytes = kv_row_bytes(lay->format, hkv);
  c.offsets = offsets;
  c.format = lay->format;
  c.hkv = hkv;
  *out = c;
  return P2P_OK;
}

}  // namespace p2p

namespace {

// The ragged rows' host-side checks (an empty call's arrays may be NULL).
p2p_status check_rows(p2p_ctx* ctx, const int32_t* past, const int32_t* row_start, int32_t nseq,
                      int64_t n_rows, int32_t max_len, const char* who) {
  if (nseq > 0 && n_rows > 0 && (!past || !row_start))
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: NULL position or row_start array", who);
  if (n_rows < 0 || n_rows > INT32_MAX || max_len < 0)
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: n_rows %lld max_len %d", who, (long long)n_rows,
                max_len);
  return P2P_OK;
}

p2p_status check_f16(p2p_ctx* ctx, const p2p_attn_params* prm, const char* who) {
  p2p_status st = p2p::ctx_check_params(ctx, prm);
  if (st == P2P_OK && prm->dtype != P2P_F16)
    return fail(ctx, P2P_ERR_UNSUPPORTED, "%s: rows must be f16", who);
  return st;
}

}  // namespace

extern "C" {

int64_t p2p_kv_q4_row_bytes(int32_t num_kv_heads) {
  return num_kv_heads > 0 ? p2p::q4_row_bytes(num_kv_heads) : 0;
}

p2p_status p2p_kv_quantize_q4(p2p_ctx* ctx, const void* src, void* dst, int64_t rows,
                              int32_t num_kv_heads, void* stream) {
  if (!ctx) return P2P_ERR_INVALID_ARG;
  if (rows == 0 && num_kv_heads > 0) return P2P_OK;
  if (!src || !dst || rows < 0 || num_kv_heads <= 0)
    return fail(ctx, P2P_ERR_INVALID_ARG, "kv_quantize_q4: NULL buffer, rows %lld or kv heads %d",
                (long long)rows, num_kv_heads);
  if (!aligned(src, 16) || !aligned(dst, 16))
    return fail(ctx, P2P_ERR_INVALID_ARG, "kv_quantize_q4: buffers must be 16-byte aligned");
  OnDevice g(p2p::ctx_device(ctx));
  return launched(ctx, p2p::launch_quantize_q4(src, dst, rows, num_kv_heads,
                                               p2p::ctx_num_sms(ctx),
                                               static_cast<cudaStream_t>(stream)),
                  "kv_quantize_q4 launch");
}

p2p_status p2p_kv_append(p2p_ctx* ctx, const p2p_attn_params* prm, const p2p_kv_layout* layout,
                         const void* qkv, int64_t ld_qkv, const void* norm_w, const void* rope,
                         void* k_cache, void* v_cache, int64_t kv_rows, const int32_t* offsets,
                         const int32_t* past, const int32_t* row_start, int32_t nseq,
                         int64_t n_rows, int32_t max_len, void* q_out, int64_t ld_q,
                         void* stream) {
  if (!ctx) return P2P_ERR_INVALID_ARG;
  p2p_status st = check_f16(ctx, prm, "kv_append");
  if (st != P2P_OK) return st;
  p2p::AppendArgs a{};
  st = p2p::make_kv_view(ctx, layout, prm->num_kv_heads, k_cache, v_cache, kv_rows, offsets, nseq,
                         "kv_append", &a.kv);
  if (st != P2P_OK) return st;
  if ((st = check_rows(ctx, past, row_start, nseq, n_rows, max_len, "kv_append")) != P2P_OK) return st;
  if (nseq == 0 || n_rows == 0) return P2P_OK;
  const int64_t qw = int64_t(prm->num_heads) * 64, row = qw + 2 * int64_t(prm->num_kv_heads) * 64;
  if (!qkv || !rope || ld_qkv < row || (q_out && ld_q < qw))
    return fail(ctx, P2P_ERR_INVALID_ARG, "kv_append: NULL buffer, ld_qkv %lld or ld_q %lld",
                (long long)ld_qkv, (long long)ld_q);
  if (!aligned(qkv, 8) || !aligned(rope, 8) || !aligned(norm_w, 8) || !aligned(q_out, 8) ||
      ld_qkv % 4 || (q_out && ld_q % 4))
    return fail(ctx, P2P_ERR_INVALID_ARG,
                "kv_append: qkv, q_out, norm_w and rope must be 8-byte aligned, ld_qkv and ld_q "
                "multiples of 4");
  if (q_out && !(q_out == qkv && (ld_q == ld_qkv || n_rows == 1)) &&
      p2p::rows_overlap(qkv, ld_qkv * 2, row * 2, q_out, ld_q * 2, qw * 2, n_rows))
    return fail(ctx, P2P_ERR_INVALID_ARG,
                "kv_append: q_out overlaps qkv (in place it starts with it and has its pitch, %lld)",
                (long long)ld_qkv);
  if ((st = p2p::ctx_check_rope(ctx, rope, max_len, "kv_append")) != P2P_OK) return st;
  a.at = {past, row_start, nseq, n_rows, max_len};
  a.qkv = static_cast<const __half*>(qkv);
  a.ld_qkv = ld_qkv;
  a.norm_w = static_cast<const __half*>(norm_w);
  a.rope = static_cast<const __half*>(rope);
  a.q_out = static_cast<__half*>(q_out);
  a.ld_q = ld_q;
  a.hq = prm->num_heads;
  a.eps = p2p::eff_eps_of(prm);
  a.err = p2p::ctx_dev_err(ctx);
  OnDevice g(p2p::ctx_device(ctx));
  return launched(ctx, p2p::launch_kv_append(a, p2p::ctx_num_sms(ctx),
                                             static_cast<cudaStream_t>(stream)),
                  "kv_append launch");
}

p2p_status p2p_kv_read(p2p_ctx* ctx, const p2p_kv_layout* layout, int32_t num_kv_heads,
                       const void* k_cache, const void* v_cache, int64_t kv_rows,
                       const int32_t* offsets, const int32_t* first, const int32_t* row_start,
                       int32_t nseq, int64_t n_rows, int32_t max_len, void* k_out, void* v_out,
                       void* stream) {
  if (!ctx) return P2P_ERR_INVALID_ARG;
  if (num_kv_heads <= 0 || num_kv_heads > 65535)
    return fail(ctx, P2P_ERR_INVALID_ARG, "kv_read: num_kv_heads %d", num_kv_heads);
  p2p::ReadArgs a{};
  p2p_status st = p2p::make_kv_view(ctx, layout, num_kv_heads, k_cache, v_cache, kv_rows, offsets,
                                    nseq, "kv_read", &a.kv);
  if (st != P2P_OK) return st;
  if ((st = check_rows(ctx, first, row_start, nseq, n_rows, max_len, "kv_read")) != P2P_OK) return st;
  if (nseq == 0 || n_rows == 0) return P2P_OK;
  if ((!k_out && !v_out) || !aligned(k_out, 16) || !aligned(v_out, 16))
    return fail(ctx, P2P_ERR_INVALID_ARG,
                "kv_read: outputs must be 16-byte aligned and not both NULL");
  a.at = {first, row_start, nseq, n_rows, max_len};
  a.k_out = static_cast<__half*>(k_out);
  a.v_out = static_cast<__half*>(v_out);
  a.err = p2p::ctx_dev_err(ctx);
  OnDevice g(p2p::ctx_device(ctx));
  return launched(ctx, p2p::launch_kv_read(a, p2p::ctx_num_sms(ctx),
                                           static_cast<cudaStream_t>(stream)),
                  "kv_read launch");
}

p2p_status p2p_attn_chunk_kv(p2p_ctx* ctx, const p2p_attn_params* prm,
                             const p2p_kv_layout* layout, const void* q, int64_t ld_q,
                             const void* k_cache, const void* v_cache, int64_t kv_rows,
                             const int32_t* offsets, const int32_t* past,
                             const int32_t* row_start, int32_t nseq, int64_t n_rows,
                             int32_t max_len, void* out, int64_t ld_o, void* stream) {
  if (!ctx) return P2P_ERR_INVALID_ARG;
  p2p_status st = check_f16(ctx, prm, "attn_chunk_kv");
  if (st != P2P_OK) return st;
  p2p::ChunkArgs a{};
  st = p2p::make_kv_view(ctx, layout, prm->num_kv_heads, k_cache, v_cache, kv_rows, offsets, nseq,
                         "attn_chunk_kv", &a.kv);
  if (st != P2P_OK) return st;
  if ((st = check_rows(ctx, past, row_start, nseq, n_rows, max_len, "attn_chunk_kv")) != P2P_OK)
    return st;
  if (nseq == 0 || n_rows == 0) return P2P_OK;
  const int64_t qw = int64_t(prm->num_heads) * 64;
  if (!q || !out || ld_q < qw || ld_o < qw)
    return fail(ctx, P2P_ERR_INVALID_ARG, "attn_chunk_kv: NULL buffer, ld_q %lld or ld_o %lld",
                (long long)ld_q, (long long)ld_o);
  if (!aligned(q, 16) || !aligned(out, 16) || ld_q % 8 || ld_o % 8)
    return fail(ctx, P2P_ERR_INVALID_ARG,
                "attn_chunk_kv: q and out must be 16-byte aligned, ld_q and ld_o multiples of 8");
  if (p2p::rows_overlap(q, ld_q * 2, qw * 2, out, ld_o * 2, qw * 2, n_rows))
    return fail(ctx, P2P_ERR_INVALID_ARG, "attn_chunk_kv: q and out overlap");
  a.at = {past, row_start, nseq, n_rows, std::min(max_len, p2p::kMaxKeys)};
  a.q = static_cast<const __half*>(q);
  a.ld_q = ld_q;
  a.out = static_cast<__half*>(out);
  a.ld_o = ld_o;
  a.hq = prm->num_heads;
  a.scale_log2 = p2p::eff_scale_log2(prm);
  a.err = p2p::ctx_dev_err(ctx);
  if (a.kv.kv_rows > (int64_t(INT32_MAX) >> a.kv.shift))
    return fail(ctx, P2P_ERR_UNSUPPORTED, "attn_chunk_kv: caches of more than 2^31 - 1 rows");
  OnDevice g(p2p::ctx_device(ctx));
  unsigned char* ws = nullptr;
  st = p2p::ctx_serve_workspace(ctx, static_cast<cudaStream_t>(stream), "attn_chunk_kv", &ws);
  if (st != P2P_OK) return st;
  a.joins = reinterpret_cast<int4*>(ws);
  a.parts = reinterpret_cast<float*>(ws + p2p::chunk_join_bytes(p2p::ctx_num_sms(ctx)));
  a.wait_deficit = p2p::debug_wait_deficit();
  return launched(ctx, p2p::launch_attn_chunk(a, p2p::ctx_num_sms(ctx),
                                              static_cast<cudaStream_t>(stream)),
                  "attn_chunk_kv launch");
}

p2p_status p2p_logits_pick(p2p_ctx* ctx, const p2p_logits* args, void* stream) {
  if (!ctx) return P2P_ERR_INVALID_ARG;
  if (!args) return fail(ctx, P2P_ERR_INVALID_ARG, "logits_pick: arguments are NULL");
  const p2p_logits& g = *args;
  if (g.dtype != P2P_F16 && g.dtype != P2P_F32)
    return fail(ctx, P2P_ERR_UNSUPPORTED, "logits_pick: dtype %d", g.dtype);
  if (g.rows == 0) return P2P_OK;
  if (!g.logits || !g.tok || g.rows < 0 || g.rows > 65535 || g.vocab <= 0 || g.ld < g.vocab ||
      (g.out && g.ld_out < g.vocab))
    return fail(ctx, P2P_ERR_INVALID_ARG,
                "logits_pick: NULL buffer, rows %d, vocab %d, ld %lld or ld_out %lld", g.rows,
                g.vocab, (long long)g.ld, (long long)g.ld_out);
  if (g.vocab > P2P_MAX_VOCAB)
    return fail(ctx, P2P_ERR_UNSUPPORTED, "logits_pick: vocab %d, at most %d", g.vocab,
                P2P_MAX_VOCAB);
  if (g.out == g.logits && g.ld != g.ld_out)
    return fail(ctx, P2P_ERR_INVALID_ARG, "logits_pick: in place with ld %lld and ld_out %lld",
                (long long)g.ld, (long long)g.ld_out);
  const unsigned es = g.dtype == P2P_F32 ? 4 : 2;
  if (!aligned(g.logits, es) || !aligned(g.out, es))
    return fail(ctx, P2P_ERR_INVALID_ARG, "logits_pick: logits not aligned to their type");
  if (g.out && g.out != g.logits &&
      p2p::rows_overlap(g.logits, g.ld * es, int64_t(g.vocab) * es, g.out, g.ld_out * es,
                        int64_t(g.vocab) * es, g.rows))
    return fail(ctx, P2P_ERR_INVALID_ARG, "logits_pick: out overlaps logits other than in place");
  if (g.hist && (!g.hist_len || g.hist_cap < 0 || g.ld_hist < g.hist_cap))
    return fail(ctx, P2P_ERR_INVALID_ARG,
                "logits_pick: hist needs hist_len and 0 <= hist_cap %d <= ld_hist %lld",
                g.hist_cap, (long long)g.ld_hist);
  if (!g.hist && (g.hist_len || g.prompt_len))
    return fail(ctx, P2P_ERR_INVALID_ARG, "logits_pick: hist_len or prompt_len without hist");
  if (g.bias_start && (g.n_bias < 0 || (g.n_bias > 0 && (!g.bias_tok || !g.bias_val))))
    return fail(ctx, P2P_ERR_INVALID_ARG, "logits_pick: bias_start needs bias_tok and bias_val");
  if (g.mask && g.ld_mask < (int64_t(g.vocab) + 31) / 32)
    return fail(ctx, P2P_ERR_INVALID_ARG, "logits_pick: ld_mask %lld for vocab %d",
                (long long)g.ld_mask, g.vocab);
  p2p::LogitsArgs a{};
  a.logits = g.logits;
  a.out = g.out;
  a.tok = g.tok;
  a.ld = g.ld;
  a.ld_out = g.ld_out;
  a.rows = g.rows;
  a.vocab = g.vocab;
  a.advance = g.advance != 0;
  a.hist = g.hist;
  a.hist_len = g.hist_len;
  a.prompt_len = g.prompt_len;
  a.past = g.past;
  a.ld_hist = g.ld_hist;
  a.hist_cap = g.hist_cap;
  a.n_bias = g.n_bias;
  a.repetition = g.repetition;
  a.presence = g.presence;
  a.frequency = g.frequency;
  a.bias_start = g.n_bias > 0 ? g.bias_start : nullptr;
  a.bias_tok = g.bias_tok;
  a.bias_val = g.bias_val;
  a.mask = g.mask;
  a.ld_mask = g.ld_mask;
  a.err = p2p::ctx_dev_err(ctx);
  OnDevice d(p2p::ctx_device(ctx));
  return launched(ctx, p2p::launch_logits_pick(a, g.dtype, static_cast<cudaStream_t>(stream)),
                  "logits_pick launch");
}

}  // extern "C"
