// C ABI of the token-side operators (declared in include/theria_sdpa.h): argument validation and launch sequencing. No
// device memory is allocated here.
#include <cmath>

#include "../../include/theria_sdpa.h"
#include "token_params.hpp"

#define THERIA_API extern "C" __attribute__((visibility("default")))

namespace theria {
namespace {

constexpr int64_t kMost = (int64_t(1) << 31) - 64;  // rows and tokens, whose 32-bit indexes are rounded up to pieces
// Rows of a table or of logits: with the workgroups that they take, a launch has to hold fewer than 2^32 threads.
constexpr int64_t kMostClasses = int64_t(1) << 27, kMostLogits = int64_t(1) << 26;

const char* check_type(int dtype) { return dtype < 0 || dtype > 2 ? "dtype must be 0 (f32), 1 (f16) or 2 (bf16)" : nullptr; }

// A view's fault, or null.
const char* check_rows(const theria_rows_t* t, bool required, int64_t rows) {
  if (!t || !t->data) return required && rows > 0 ? "a required matrix is absent" : nullptr;
  return t->stride_row < 0 ? "a matrix has a negative stride" : nullptr;
}

Rows in(const theria_rows_t* t) { return t ? Rows{t->data, t->stride_row} : Rows{nullptr, 0}; }
MutRows out(const theria_rows_t* t) { return t ? MutRows{t->data, t->stride_row} : MutRows{nullptr, 0}; }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

#define THERIA_CHECK(expr)                                        \
  do {                                                            \
    if (const char* m_ = (expr)) return fail(THERIA_ERR_CONTRACT, m_); \
  } while (0)
#define THERIA_NEED(ok, msg)                                \
  do {                                                      \
    if (!(ok)) return fail(THERIA_ERR_CONTRACT, msg);       \
  } while (0)

const char* norm_from(const theria_layer_norm_problem_t* p, NormParams& n) {
  if (!p) return "problem is required";
  if (const char* m = check_type(p->dtype)) return m;
  if (p->param_dtype != p->dtype && p->param_dtype != 0) return "param_dtype must be dtype or float32";
  if (p->width < 1 || p->width > kNormMaxWidth) return "width must be in 1..16384";
  if (p->rows < 0 || p->rows > kMost) return "rows must be in 0..2^31 - 64";
  if (!(p->eps >= 0.f) || std::isinf(p->eps)) return "eps must be finite and not negative";
  n = NormParams{};
  n.dtype = p->dtype;
  n.param_dtype = p->param_dtype;
  n.rows = p->rows;
  n.width = p->width;
  n.eps = p->eps;
  return nullptr;
}

const char* embed_from(const theria_embedding_problem_t* p, EmbedParams& e) {
  if (!p) return "problem is required";
  if (const char* m = check_type(p->dtype)) return m;
  if (p->width < 1 || p->width > (1 << 20)) return "width must be in 1..2^20";
  if (p->n < 0 || p->n > kMost || p->classes < 0 || p->classes > kMostClasses) return "n must be in 0..2^31 - 64 and classes in 0..2^27";
  if (p->padding < -1 || p->padding >= p->classes) return "padding must be -1 or a row of the table";
  if (!std::isfinite(p->scale)) return "scale must be finite";
  e = EmbedParams{};
  e.dtype = p->dtype;
  e.ids64 = p->ids64 != 0;
  e.n = p->n;
  e.classes = p->classes;
  e.width = p->width;
  e.scale = p->scale;
  e.padding = p->padding;
  return nullptr;
}

const char* ce_from(const theria_linear_ce_problem_t* p, CeParams& c) {
  if (!p) return "problem is required";
  if (const char* m = check_type(p->dtype)) return m;
  if (p->reduction < 0 || p->reduction > 2) return "reduction must be 0 (none), 1 (mean) or 2 (sum)";
  if (p->width < 1 || p->width > (1 << 20)) return "width must be in 1..2^20";
  if (p->n < 0 || p->n > kMostLogits) return "n must be in 0..2^26";
  if (p->classes < 1 || p->classes > kMostLogits) return "classes must be in 1..2^26";
  c = CeParams{};
  c.dtype = p->dtype;
  c.target64 = p->target64 != 0;
  c.reduction = p->reduction;
  c.n = p->n;
  c.classes = p->classes;
  c.ignore = p->ignore;
  c.width = p->width;
  return nullptr;
}

const char* ce_inputs(const theria_linear_ce_problem_t* p, CeParams& c, const theria_rows_t* x, const theria_rows_t* w, const void* bias,
                      const void* target, const float* stats, const void* ws) {
  if (const char* m = ce_from(p, c)) return m;
  if (const char* m = check_rows(x, true, c.n)) return m;
  if (const char* m = check_rows(w, true, c.classes)) return m;
  if (c.n > 0 && (!target || !stats)) return "target and stats are required";
  if (!ws || reinterpret_cast<uintptr_t>(ws) % 256) return "a 256-byte-aligned workspace is required";
  c.x = in(x);
  c.w = in(w);
  c.bias = bias;
  c.target = target;
  c.stats = const_cast<float*>(stats);
  c.ws = const_cast<void*>(ws);
  return nullptr;
}

}  // namespace
}  // namespace theria

using namespace theria;

THERIA_API int theria_layer_norm_fwd(const theria_layer_norm_problem_t* p, const theria_rows_t* x, const void* weight, const void* bias,
                                     const theria_rows_t* y, float* mean, float* rstd, void* stream) {
  NormParams n;
  THERIA_CHECK(norm_from(p, n));
  THERIA_CHECK(check_rows(x, true, n.rows));
  THERIA_CHECK(check_rows(y, true, n.rows));
  THERIA_NEED(n.rows == 0 || (mean && rstd), "mean and rstd are required");
  if (n.rows == 0) return THERIA_OK;
  n.x = in(x), n.y = out(y);
  n.weight = weight, n.bias = bias, n.mean = mean, n.rstd = rstd;
  return hip_status(launch_norm_fwd(n, (hipStream_t)stream), "theria_layer_norm_fwd");
}

THERIA_API int64_t theria_layer_norm_ws_floats(const theria_layer_norm_problem_t* p) {
  NormParams n;
  return norm_from(p, n) ? 0 : norm_ws_floats(n);
}

THERIA_API int theria_layer_norm_bwd(const theria_layer_norm_problem_t* p, const theria_rows_t* x, const void* weight,
                                     const theria_rows_t* dout, const float* mean, const float* rstd, const theria_rows_t* dx,
                                     void* dweight, void* dbias, float* ws, void* stream) {
  NormParams n;
  THERIA_CHECK(norm_from(p, n));
  THERIA_NEED(n.rows > 0, "rows must be positive (no rows: the gradients are zeros)");
  THERIA_CHECK(check_rows(x, true, n.rows));
  THERIA_CHECK(check_rows(dout, true, n.rows));
  THERIA_CHECK(check_rows(dx, false, n.rows));
  THERIA_NEED(mean && rstd, "mean and rstd are required");
  THERIA_NEED(ws || !(dweight || dbias), "a workspace is required for dweight and dbias");
  n.x = in(x), n.dout = in(dout), n.dx = out(dx);
  n.weight = weight, n.mean = const_cast<float*>(mean), n.rstd = const_cast<float*>(rstd);
  n.dw = dweight, n.db = dbias, n.ws = ws;
  if (!n.dx.p && !dweight && !dbias) return THERIA_OK;
  return hip_status(launch_norm_bwd(n, (hipStream_t)stream), "theria_layer_norm_bwd");
}

THERIA_API int theria_layer_norm_bwd_bwd(const theria_layer_norm_problem_t* p, const theria_rows_t* x, const void* weight,
                                         const theria_rows_t* dout, const float* mean, const float* rstd, const theria_rows_t* gdx,
                                         const void* gdw, const void* gdb, const theria_rows_t* out_gx, void* out_gw,
                                         const theria_rows_t* out_gdout, float* ws, void* stream) {
  NormParams n;
  THERIA_CHECK(norm_from(p, n));
  THERIA_NEED(n.rows > 0, "rows must be positive (no rows: the gradients are zeros)");
  THERIA_CHECK(check_rows(x, true, n.rows));
  THERIA_CHECK(check_rows(dout, true, n.rows));
  THERIA_CHECK(check_rows(gdx, false, n.rows));
  THERIA_CHECK(check_rows(out_gx, false, n.rows));
  THERIA_CHECK(check_rows(out_gdout, false, n.rows));
  THERIA_NEED(mean && rstd, "mean and rstd are required");
  THERIA_NEED(ws || !out_gw, "a workspace is required for out_gw");
  n.x = in(x), n.dout = in(dout), n.gdx = in(gdx);
  n.weight = weight, n.gdw = gdw, n.gdb = gdb;
  n.mean = const_cast<float*>(mean), n.rstd = const_cast<float*>(rstd);
  n.out_gx = out(out_gx), n.out_gdout = out(out_gdout), n.out_gw = out_gw, n.ws = ws;
  if (!n.out_gx.p && !n.out_gdout.p && !out_gw) return THERIA_OK;
  return hip_status(launch_norm_bwd_bwd(n, (hipStream_t)stream), "theria_layer_norm_bwd_bwd");
}

THERIA_API int theria_embedding_fwd(const theria_embedding_problem_t* p, const void* ids, const theria_rows_t* table,
                                    int32_t zero_padding, const theria_rows_t* o, void* stream) {
  EmbedParams e;
  THERIA_CHECK(embed_from(p, e));
  THERIA_CHECK(check_rows(table, true, e.n > 0 ? e.classes : 0));
  THERIA_CHECK(check_rows(o, true, e.n));
  THERIA_NEED(e.n == 0 || ids, "ids are required");
  if (e.n == 0) return THERIA_OK;
  e.ids = ids, e.table = in(table), e.out = out(o), e.zero_padding = zero_padding != 0;
  return hip_status(launch_embed_fwd(e, (hipStream_t)stream), "theria_embedding_fwd");
}

THERIA_API int64_t theria_embedding_ws_bytes(const theria_embedding_problem_t* p) {
  EmbedParams e;
  return embed_from(p, e) ? 0 : embed_ws_bytes(e);
}

THERIA_API int theria_embedding_bwd(const theria_embedding_problem_t* p, const void* ids, const theria_rows_t* dout,
                                    const theria_rows_t* dtable, void* ws, void* stream) {
  EmbedParams e;
  THERIA_CHECK(embed_from(p, e));
  THERIA_CHECK(check_rows(dout, true, e.n));
  THERIA_CHECK(check_rows(dtable, true, e.classes));
  THERIA_NEED(e.n == 0 || (ids && ws && aligned16(ws)), "ids and a 16-byte-aligned workspace are required");
  if (e.classes == 0) return THERIA_OK;
  e.ids = ids, e.dout = in(dout), e.out = out(dtable), e.ws = ws;
  return hip_status(launch_embed_bwd(e, (hipStream_t)stream), "theria_embedding_bwd");
}

THERIA_API int64_t theria_linear_ce_ws_bytes(const theria_linear_ce_problem_t* p, const theria_rows_t* weight, int32_t backward,
                                             int32_t need_dx, int32_t need_dweight, int32_t need_dbias) {
  CeParams c;
  if (ce_from(p, c) || !weight) return 0;
  c.w = in(weight);
  c.dx.p = need_dx ? weight->data : nullptr;  // the layout asks only whether they are wanted
  c.dw.p = need_dweight ? weight->data : nullptr;
  c.db = need_dbias ? weight->data : nullptr;
  return ce_ws_bytes(c, backward != 0);
}

THERIA_API int theria_linear_ce_fwd(const theria_linear_ce_problem_t* p, const theria_rows_t* x, const theria_rows_t* weight,
                                    const void* bias, const void* target, float* loss, float* stats, void* ws, void* stream) {
  CeParams c;
  THERIA_CHECK(ce_inputs(p, c, x, weight, bias, target, stats, ws));
  THERIA_NEED(loss || (c.reduction == kCeNone && c.n == 0), "loss is required");
  if (c.reduction == kCeNone && c.n == 0) return THERIA_OK;
  c.loss = loss;
  return hip_status(launch_ce_fwd(c, (hipStream_t)stream), "theria_linear_ce_fwd");
}

THERIA_API int theria_linear_ce_bwd(const theria_linear_ce_problem_t* p, const theria_rows_t* x, const theria_rows_t* weight,
                                    const void* bias, const void* target, const float* stats, const float* dloss,
                                    const theria_rows_t* dx, const theria_rows_t* dweight, void* dbias, void* ws, void* stream) {
  CeParams c;
  THERIA_CHECK(ce_inputs(p, c, x, weight, bias, target, stats, ws));
  THERIA_CHECK(check_rows(dx, false, c.n));
  THERIA_CHECK(check_rows(dweight, false, c.classes));
  THERIA_NEED(dloss || (c.reduction == kCeNone && c.n == 0), "dloss is required");
  c.gout = dloss;
  c.dx = out(dx), c.dw = out(dweight), c.db = dbias;
  if (!c.dx.p && !c.dw.p && !dbias) return THERIA_OK;
  return hip_status(launch_ce_bwd(c, (hipStream_t)stream), "theria_linear_ce_bwd");
}
