// q8_api.cu -- the C entry points of the 8-bit layer operators (rows with a scale each, the norm in
// front of them, their products).  Host-side checks only.
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdarg>
#include <cstdio>

// The library is built with -fvisibility=hidden; only the declared C ABI is exported.
#pragma GCC visibility push(default)
#include "../../include/p2p_attn.h"
#pragma GCC visibility pop
#include "host_internal.h"
#include "kernels.h"
#include "rows.h"

static_assert(P2P_ACT_SILU == p2p::kActSilu && P2P_ACT_GELU == p2p::kActGelu, "activations");
static_assert(P2P_F16 == 0 && P2P_F32 == 1, "the launchers' types");

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
  explicit OnDevice(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) cudaSetDevice(dev);
    else prev = -1;
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

p2p_status launched(p2p_ctx* ctx, cudaError_t e, const char* who) {
  if (e == cudaSuccess) return P2P_OK;
  cudaGetLastError();
  return fail(ctx, P2P_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}

// Rows of a call: n of them, `width` bytes each, `pitch` bytes apart.
struct Span {
  const void* p;
  int64_t pitch, width, n;
  const char* name;
};

Span rows_of(const p2p_q8_rows* r, const char* name) { return {r->q, r->ld, r->cols, r->rows, name}; }
Span scales_of(const p2p_q8_rows* r, const char* name) {
  return {r->scale, 0, 4 * int64_t(r->rows), 1, name};
}

bool meet(const Span& a, const Span& b) {
  if (!a.p || !b.p || a.n <= 0 || b.n <= 0 || a.width <= 0 || b.width <= 0) return false;
  if (a.n == b.n) return p2p::rows_overlap(a.p, a.pitch, a.width, b.p, b.pitch, b.width, a.n);
  // different counts: the ranges they span
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  return pa < pb + uintptr_t((b.n - 1) * b.pitch + b.width) &&
         pb < pa + uintptr_t((a.n - 1) * a.pitch + a.width);
}

// `out` against the spans behind it.
p2p_status apart(p2p_ctx* ctx, const char* who, const Span& out, std::initializer_list<Span> others) {
  for (const Span& o : others)
    if (meet(out, o))
      return fail(ctx, P2P_ERR_INVALID_ARG, "%s: %s overlaps %s", who, out.name, o.name);
  return P2P_OK;
}

p2p_status check_dtype(p2p_ctx* ctx, int32_t dtype, const char* who) {
  if (dtype != P2P_F16 && dtype != P2P_F32)
    return fail(ctx, P2P_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  return P2P_OK;
}

p2p_status check_q8(p2p_ctx* ctx, const p2p_q8_rows* r, const char* name, const char* who) {
  if (!r) return fail(ctx, P2P_ERR_INVALID_ARG, "%s: %s is NULL", who, name);
  if (r->rows < 0 || r->rows > P2P_MAX_Q8_ROWS || r->cols < 1 || r->cols > P2P_MAX_Q8_COLS)
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: %s has %d rows (0..%d) of %d codes (1..%d)", who, name,
                r->rows, P2P_MAX_Q8_ROWS, r->cols, P2P_MAX_Q8_COLS);
  if (r->rows == 0) return P2P_OK;
  if (!r->q || !r->scale)
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: %s has no codes or no scales", who, name);
  if (!aligned(r->q, 16) || r->ld % 16 || r->ld < r->cols || !aligned(r->scale, 4))
    return fail(ctx, P2P_ERR_INVALID_ARG,
                "%s: %s: codes 16-byte aligned, ld %lld a multiple of 16 and at least %d, scales 4-byte "
                "aligned",
                who, name, (long long)r->ld, r->cols);
  return P2P_OK;
}

// Values of `type` bytes, `rows` rows of `cols`.
p2p_status check_rows(p2p_ctx* ctx, const void* p, int64_t ld, int64_t cols, unsigned type,
                      const char* name, const char* who) {
  if (!p || ld < cols || !aligned(p, type))
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: %s is NULL, not aligned to its type, or ld %lld < %lld",
                who, name, (long long)ld, (long long)cols);
  return P2P_OK;
}

p2p::Q8Rows view(const p2p_q8_rows* r) {
  return {static_cast<int8_t*>(r->q), r->scale, r->ld, r->rows, r->cols};
}

}  // namespace

extern "C" {

p2p_status p2p_quantize_rows_q8(p2p_ctx* ctx, const p2p_quantize_rows* args, void* stream) {
  if (!ctx) return P2P_ERR_INVALID_ARG;
  const char* who = "quantize_rows_q8";
  if (!args) return fail(ctx, P2P_ERR_INVALID_ARG, "%s: arguments are NULL", who);
  const void* src = args->src;
  const int64_t ld_src = args->ld_src;
  const int32_t dtype = args->dtype;
  const p2p_q8_rows* dst = &args->dst;
  p2p_status st;
  if ((st = check_dtype(ctx, dtype, who)) != P2P_OK) return st;
  if ((st = check_q8(ctx, dst, "dst", who)) != P2P_OK) return st;
  if (dst->rows == 0) return P2P_OK;
  const unsigned es = dtype == P2P_F32 ? 4 : 2;
  if ((st = check_rows(ctx, src, ld_src, dst->cols, es, "src", who)) != P2P_OK) return st;
  const Span in{src, ld_src * es, int64_t(dst->cols) * es, dst->rows, "src"};
  const Span codes = rows_of(dst, "dst's codes"), scales = scales_of(dst, "dst's scales");
  if ((st = apart(ctx, who, codes, {in, scales})) != P2P_OK) return st;
  if ((st = apart(ctx, who, scales, {in})) != P2P_OK) return st;
  p2p::RowsQ8Args a{};
  a.x = src;
  a.ld_x = ld_src;
  a.out = view(dst);
  OnDevice g(p2p::ctx_device(ctx));
  return launched(ctx, p2p::launch_rows_q8(a, dtype, p2p::ctx_num_sms(ctx),
                                           static_cast<cudaStream_t>(stream)),
                  who);
}

p2p_status p2p_read_rows_q8(p2p_ctx* ctx, const p2p_read_rows* args, void* stream) {
  if (!ctx) return P2P_ERR_INVALID_ARG;
  const char* who = "read_rows_q8";
  if (!args) return fail(ctx, P2P_ERR_INVALID_ARG, "%s: arguments are NULL", who);
  const p2p_q8_rows* src = &args->src;
  const int32_t* index = args->index;
  const int64_t rows = args->rows, ld_out = args->ld_out;
  const int32_t dtype = args->dtype;
  void* out = args->out;
  p2p_status st;
  if ((st = check_dtype(ctx, dtype, who)) != P2P_OK) return st;
  if ((st = check_q8(ctx, src, "src", who)) != P2P_OK) return st;
  if (rows < 0 || rows > P2P_MAX_Q8_ROWS || (!index && rows > src->rows) || !aligned(index, 4))
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: %lld rows of %d, index %p", who, (long long)rows,
                src->rows, (const void*)index);
  if (rows == 0) return P2P_OK;
  // a row of zeros times an infinity would be NaN
  if (!(args->factor >= -FLT_MAX && args->factor <= FLT_MAX))
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: factor %g", who, double(args->factor));
  const unsigned es = dtype == P2P_F32 ? 4 : 2;
  if ((st = check_rows(ctx, out, ld_out, src->cols, es, "out", who)) != P2P_OK) return st;
  const Span to{out, ld_out * es, int64_t(src->cols) * es, rows, "out"};
  if ((st = apart(ctx, who, to, {rows_of(src, "src's codes"), scales_of(src, "src's scales"),
                                 {index, 0, 4 * rows, 1, "index"}})) != P2P_OK)
    return st;
  const p2p::ReadQ8Args a{view(src), index, rows, args->factor == 0.f ? 1.f : args->factor, out, ld_out, p2p::ctx_dev_err(ctx)};
  OnDevice g(p2p::ctx_device(ctx));
  return launched(ctx, p2p::launch_read_q8(a, dtype, static_cast<cudaStream_t>(stream)), who);
}

p2p_status p2p_add_norm_q8(p2p_ctx* ctx, const p2p_add_norm* args, void* stream) {
  if (!ctx) return P2P_ERR_INVALID_ARG;
  const char* who = "add_norm_q8";
  if (!args) return fail(ctx, P2P_ERR_INVALID_ARG, "%s: arguments are NULL", who);
  const p2p_add_norm& g = *args;
  p2p_status st;
  if ((st = check_dtype(ctx, g.dtype, who)) != P2P_OK) return st;
  const int32_t rows = g.out.rows, cols = g.out.cols;
  if (g.out.q) {
    if ((st = check_q8(ctx, &g.out, "out", who)) != P2P_OK) return st;
  } else if (rows < 0 || rows > P2P_MAX_Q8_ROWS || cols < 1 || cols > P2P_MAX_Q8_COLS) {
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: %d rows (0..%d) of %d values (1..%d)", who, rows,
                P2P_MAX_Q8_ROWS, cols, P2P_MAX_Q8_COLS);
  }
  if (rows == 0) return P2P_OK;
  if (!g.sum && !g.y && !g.out.q)
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: sum, y and out.q are all NULL", who);
  if (!(g.eps >= 0.f && g.eps <= 3.4e38f))
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: eps %g", who, double(g.eps));
  const unsigned es = g.dtype == P2P_F32 ? 4 : 2;
  if ((st = check_rows(ctx, g.x, g.ld_x, cols, es, "x", who)) != P2P_OK) return st;
  if (g.residual && (st = check_rows(ctx, g.residual, g.ld_r, cols, es, "residual", who)) != P2P_OK)
    return st;
  if (g.sum && (st = check_rows(ctx, g.sum, g.ld_sum, cols, es, "sum", who)) != P2P_OK) return st;
  if (g.y && (st = check_rows(ctx, g.y, g.ld_y, cols, es, "y", who)) != P2P_OK) return st;
  if (!aligned(g.weight, 2))
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: weight not aligned to its type", who);
  const int64_t width = int64_t(cols) * es;
  const Span none{nullptr, 0, 0, 0, ""};
  const Span x{g.x, g.ld_x * es, width, rows, "x"}, r{g.residual, g.ld_r * es, width, rows, "residual"};
  const Span w{g.weight, 0, int64_t(cols) * 2, 1, "weight"};
  const Span sum{g.sum, g.ld_sum * es, width, rows, "sum"}, y{g.y, g.ld_y * es, width, rows, "y"};
  const Span codes = g.out.q ? rows_of(&g.out, "out's codes") : none;
  const Span scales = g.out.q ? scales_of(&g.out, "out's scales") : none;
  // in place: the same rows, element by element
  const auto same = [&](const Span& a, const Span& b) {
    return a.p == b.p && (a.pitch == b.pitch || rows == 1);
  };
  for (const Span& o : {sum, y}) {
    if (!o.p) continue;
    for (const Span& i : {x, r})
      if (!same(o, i) && meet(o, i))
        return fail(ctx, P2P_ERR_INVALID_ARG, "%s: %s overlaps %s other than in place", who, o.name,
                    i.name);
    if ((st = apart(ctx, who, o, {w, codes, scales})) != P2P_OK) return st;
  }
  if ((st = apart(ctx, who, sum, {y})) != P2P_OK) return st;
  if ((st = apart(ctx, who, codes, {x, r, w, scales})) != P2P_OK) return st;
  if ((st = apart(ctx, who, scales, {x, r, w})) != P2P_OK) return st;
  p2p::RowsQ8Args a{};
  a.x = g.x;
  a.r = g.residual;
  a.w = static_cast<const __half*>(g.weight);
  a.sum = g.sum;
  a.y = g.y;
  a.out = view(&g.out);
  a.ld_x = g.ld_x;
  a.ld_r = g.ld_r;
  a.ld_sum = g.ld_sum;
  a.ld_y = g.ld_y;
  a.eps = g.eps == 0.f ? 1e-5f : g.eps;
  a.norm = 1;
  OnDevice d(p2p::ctx_device(ctx));
  return launched(ctx, p2p::launch_rows_q8(a, g.dtype, p2p::ctx_num_sms(ctx),
                                           static_cast<cudaStream_t>(stream)),
                  who);
}

p2p_status p2p_gemm_q8(p2p_ctx* ctx, const p2p_product* args, void* stream) {
  if (!ctx) return P2P_ERR_INVALID_ARG;
  const char* who = "gemm_q8";
  if (!args) return fail(ctx, P2P_ERR_INVALID_ARG, "%s: arguments are NULL", who);
  const p2p_q8_rows *w = &args->w, *x = &args->x;
  const float* bias = args->bias;
  const void* residual = args->residual;
  void* y = args->y;
  const int64_t ld_r = args->ld_r, ld_y = args->ld_y;
  const int32_t dtype = args->dtype;
  p2p_status st;
  if ((st = check_dtype(ctx, dtype, who)) != P2P_OK) return st;
  if ((st = check_q8(ctx, w, "w", who)) != P2P_OK) return st;
  if ((st = check_q8(ctx, x, "x", who)) != P2P_OK) return st;
  if (w->cols != x->cols)
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: rows of %d and %d codes", who, w->cols, x->cols);
  if (w->rows == 0 || x->rows == 0) return P2P_OK;
  const unsigned es = dtype == P2P_F32 ? 4 : 2;
  if ((st = check_rows(ctx, y, ld_y, w->rows, es, "y", who)) != P2P_OK) return st;
  if (residual && (st = check_rows(ctx, residual, ld_r, w->rows, es, "residual", who)) != P2P_OK)
    return st;
  if (!aligned(bias, 4))
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: bias not aligned to its type", who);
  const int64_t width = int64_t(w->rows) * es;
  const Span out{y, ld_y * es, width, x->rows, "y"};
  const Span res{residual, ld_r * es, width, x->rows, "residual"};
  if (!(residual == y && (ld_r == ld_y || x->rows == 1)) && meet(out, res))
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: y overlaps residual other than in place", who);
  if ((st = apart(ctx, who, out, {rows_of(w, "w's codes"), scales_of(w, "w's scales"),
                                  rows_of(x, "x's codes"), scales_of(x, "x's scales"),
                                  {bias, 0, 4 * int64_t(w->rows), 1, "bias"}})) != P2P_OK)
    return st;
  p2p::GemmQ8Args a{};
  a.x = view(x);
  a.w = view(w);
  a.bias = bias;
  a.res = residual;
  a.ld_res = ld_r;
  a.y = y;
  a.ld_y = ld_y;
  a.err = p2p::ctx_dev_err(ctx);
  a.wait_deficit = p2p::debug_wait_deficit();
  OnDevice g(p2p::ctx_device(ctx));
  return launched(ctx, p2p::launch_gemm_q8(a, dtype, p2p::ctx_num_sms(ctx),
                                           static_cast<cudaStream_t>(stream)),
                  who);
}

p2p_status p2p_gate_q8(p2p_ctx* ctx, const p2p_gated* args, void* stream) {
  if (!ctx) return P2P_ERR_INVALID_ARG;
  const char* who = "gate_q8";
  if (!args) return fail(ctx, P2P_ERR_INVALID_ARG, "%s: arguments are NULL", who);
  const p2p_q8_rows *gate = &args->gate, *up = &args->up, *x = &args->x;
  void* h = args->h;
  const int64_t ld_h = args->ld_h;
  const int32_t act = args->act;
  p2p_status st;
  if (act != P2P_ACT_SILU && act != P2P_ACT_GELU)
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: act %d", who, act);
  if ((st = check_q8(ctx, gate, "gate", who)) != P2P_OK) return st;
  if ((st = check_q8(ctx, up, "up", who)) != P2P_OK) return st;
  if ((st = check_q8(ctx, x, "x", who)) != P2P_OK) return st;
  if (gate->rows != up->rows || gate->cols != up->cols || gate->cols != x->cols)
    return fail(ctx, P2P_ERR_INVALID_ARG, "%s: gate [%d][%d], up [%d][%d], x rows of %d codes", who,
                gate->rows, gate->cols, up->rows, up->cols, x->cols);
  if (gate->rows == 0 || x->rows == 0) return P2P_OK;
  if ((st = check_rows(ctx, h, ld_h, gate->rows, 2, "h", who)) != P2P_OK) return st;
  const Span out{h, ld_h * 2, int64_t(gate->rows) * 2, x->rows, "h"};
  if ((st = apart(ctx, who, out, {rows_of(gate, "gate's codes"), scales_of(gate, "gate's scales"),
                                  rows_of(up, "up's codes"), scales_of(up, "up's scales"),
                                  rows_of(x, "x's codes"), scales_of(x, "x's scales")})) != P2P_OK)
    return st;
  p2p::GemmQ8Args a{};
  a.x = view(x);
  a.w = view(gate);
  a.up = view(up);
  a.act = act;
  a.y = h;
  a.ld_y = ld_h;
  a.err = p2p::ctx_dev_err(ctx);
  a.wait_deficit = p2p::debug_wait_deficit();
  OnDevice g(p2p::ctx_device(ctx));
  return launched(ctx, p2p::launch_gemm_q8(a, P2P_F16, p2p::ctx_num_sms(ctx),
                                           static_cast<cudaStream_t>(stream)),
                  who);
}

}  // extern "C"
