// Python binding of the hot C ABI entry points (theria_sdpa_fwd, _bwd, _jvp, _bwd_bwd, and the token-side operators)
// for torch tensors.
//
// The autograd operator calls these once per forward, backward, JVP and double backward. Building the
// theria_tensor_t views, the output tensors and the stream handle here costs about a microsecond per call,
// against ~3 us per tensor view through ctypes from Python (a double backward passes fifteen). The semantics are
// those of theria_amd/_ops.py (same argument meaning, same output dtypes, same error types): shape and device
// mismatches raise AssertionError, as the reference's guards do (theria/attention/triton_sdpa_backward.py:23-103),
// and the C ABI's own contract errors keep their status (THERIA_ERR_CONTRACT -> AssertionError,
// THERIA_ERR_HIP -> RuntimeError). Dtype and 4-D checks of the primary inputs stay in Python
// (_ops.check_inputs), which runs once per autograd operator.
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <optional>
#include <string>

#include "theria_sdpa.h"

namespace py = pybind11;

namespace {

using OptT = std::optional<at::Tensor>;

[[noreturn]] void raise_assertion(const std::string& msg) {
  PyErr_SetString(PyExc_AssertionError, msg.c_str());
  throw py::error_already_set();
}

void need(bool ok, const char* msg) {
  if (!ok) raise_assertion(msg);
}

void check_rc(int rc, const char* what) {
  if (rc == THERIA_OK) return;
  std::string msg = std::string(what) + ": " + theria_last_error();
  if (rc == THERIA_ERR_CONTRACT) raise_assertion(msg);
  PyErr_SetString(PyExc_RuntimeError, msg.c_str());
  throw py::error_already_set();
}

// The tensor a torch.func wrapper holds (SDPAOp.jvp receives its saved tensors wrapped under torch.func.jvp).
// A wrapper has no storage of its own; such calls are rare, so torch's own Python helpers unwrap it. The helpers
// are looked up once and deliberately never released: a static py::object would be destroyed after the
// interpreter has shut down, and its reference-count decrement would then crash the process at exit.
at::Tensor plain(const at::Tensor& t) {
  if (t.has_storage()) return t;
  static py::object* is_wrapped = nullptr;
  static py::object* unwrap = nullptr;
  if (!unwrap) {
    const py::object ft = py::module_::import("torch._C._functorch");
    is_wrapped = new py::object(ft.attr("is_functorch_wrapped_tensor"));
    unwrap = new py::object(ft.attr("get_unwrapped"));
  }
  at::Tensor cur = t;
  while (!cur.has_storage() && (*is_wrapped)(cur).cast<bool>()) cur = (*unwrap)(cur).cast<at::Tensor>();
  return cur;
}

// The kernels need a contiguous last dimension; any other strides (broadcast rows included) are fine.
at::Tensor rowmajor(at::Tensor t) {
  t = plain(t);
  if (t.size(-1) > 1 && t.stride(-1) != 1) t = t.contiguous();
  return t;
}

// A (B, H, rows, D) operand in the compute dtype on q's device.
at::Tensor like_rows(const at::Tensor& t_in, const at::Tensor& q, int64_t rows, const char* msg) {
  const at::Tensor t = plain(t_in);
  need(t.dim() == 4 && t.size(0) == q.size(0) && t.size(1) == q.size(1) && t.size(2) == rows &&
           t.size(3) == q.size(3) && t.device() == q.device(),
       msg);
  return rowmajor(t.scalar_type() == q.scalar_type() ? t : t.to(q.scalar_type()));
}

OptT like_rows(const OptT& t, const at::Tensor& q, int64_t rows, const char* msg) {
  if (!t) return std::nullopt;
  return like_rows(*t, q, rows, msg);
}

at::Tensor rowstat(const at::Tensor& t, const at::Tensor& q, const char* msg) {
  need(t.scalar_type() == at::kFloat && t.numel() == q.size(0) * q.size(1) * q.size(2) && t.device() == q.device(),
       msg);
  return plain(t).contiguous();
}

// Views and pointers are taken from the plain tensor: under a torch.func transform the outputs allocated here are
// wrappers too (at::empty returns one), and they are returned as such while the kernels write the storage.
theria_tensor_t view(const at::Tensor& t_in) {
  const at::Tensor t = plain(t_in);
  return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}
theria_tensor_t view(const OptT& t) { return t ? view(*t) : theria_tensor_t{nullptr, 0, 0, 0}; }
float* fptr(const at::Tensor& t) { return plain(t).data_ptr<float>(); }
float* fptr(const OptT& t) { return t ? fptr(*t) : nullptr; }

int32_t dtype_code(at::ScalarType st) {
  switch (st) {
    case at::kFloat: return THERIA_DTYPE_F32;
    case at::kHalf: return THERIA_DTYPE_F16;
    case at::kBFloat16: return THERIA_DTYPE_BF16;
    default: raise_assertion(std::string("Unsupported dtype: ") + c10::toString(st));
  }
}

theria_sdpa_problem_t problem(const at::Tensor& q, const at::Tensor& k, double scale, bool causal) {
  return {dtype_code(q.scalar_type()), (int32_t)q.size(0), (int32_t)q.size(1), (int32_t)q.size(2),
          (int32_t)k.size(2),           (int32_t)q.size(3), (float)scale,       causal ? 1 : 0};
}

void* stream_of(const at::Tensor& q) { return c10::hip::getCurrentHIPStream(q.get_device()).stream(); }

// (q, k, v) in row-major layout with matching shapes (dtype and rank were checked in Python).
void kv_shapes(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
  need(k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3),
       "k must have shape (B,H,M,D) with D matching q");
  need(v.size(0) == q.size(0) && v.size(1) == q.size(1) && v.size(2) == k.size(2) && v.size(3) == q.size(3),
       "v must have shape (B,H,M,D) matching k");
  need(k.device() == q.device() && v.device() == q.device(), "q, k and v must be on one device");
}

py::tuple fwd(at::Tensor q, at::Tensor k, at::Tensor v, double scale, bool causal, bool out_fp32, bool stats) {
  q = rowmajor(q), k = rowmajor(k), v = rowmajor(v);
  kv_shapes(q, k, v);
  const c10::hip::HIPGuard guard(q.get_device());
  const auto o = at::empty(q.sizes(), q.options().dtype(out_fp32 ? at::kFloat : q.scalar_type()));
  const auto f = q.options().dtype(at::kFloat);
  const auto lse = at::empty({q.size(0), q.size(1), q.size(2)}, f);
  OptT m, l;
  if (stats) m = at::empty_like(lse), l = at::empty_like(lse);
  const auto p = problem(q, k, scale, causal);
  const auto tq = view(q), tk = view(k), tv = view(v), to = view(o);
  // workspace of a forward whose keys are split over workgroups, on the stream that uses it
  const int64_t nws = theria_sdpa_fwd_ws_floats(&p);
  const OptT ws = nws > 0 ? OptT(at::empty({nws}, f)) : std::nullopt;
  check_rc(theria_sdpa_fwd_ws(&p, &tq, &tk, &tv, &to, out_fp32 ? 1 : 0, fptr(lse), fptr(m), fptr(l), fptr(ws), nws,
                              stream_of(q)),
           "theria_sdpa_fwd");
  return py::make_tuple(o, lse, m ? py::cast(*m) : py::none(), l ? py::cast(*l) : py::none());
}

// dQ, dK, dV and the row term, as _ops.bwd. out: (dq, dk, dv) to write instead of new tensors.
py::tuple bwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor o, const at::Tensor& lse_in,
              const at::Tensor& dout_in, double scale, bool causal, bool need_dq, bool need_dk,
              const std::optional<std::vector<at::Tensor>>& out) {
  q = rowmajor(q), k = rowmajor(k), v = rowmajor(v);
  kv_shapes(q, k, v);
  const int64_t T = q.size(2), M = k.size(2);
  const auto dout = like_rows(dout_in, q, T, "dout must have shape (B,H,T,D)");
  o = rowmajor(o);
  need(o.dim() == 4 && o.sizes() == q.sizes(), "o must have shape (B,H,T,D)");
  const bool o_f32 = o.scalar_type() == at::kFloat && q.scalar_type() != at::kFloat;
  if (!o_f32 && o.scalar_type() != q.scalar_type()) o = o.to(q.scalar_type());
  const auto lse = rowstat(lse_in, q, "lse must be a float32 (B,H,T) tensor on q's device");
  const c10::hip::HIPGuard guard(q.get_device());
  const auto delta = at::empty({q.size(0), q.size(1), T}, q.options().dtype(at::kFloat));
  OptT dq, dk;
  at::Tensor dv;
  if (out) {
    need(out->size() == 3, "out must hold (dq, dk, dv)");
    const int64_t rows[3] = {T, M, M};
    for (int i = 0; i < 3; ++i) {
      const auto& t = (*out)[i];
      need(t.dim() == 4 && t.size(0) == q.size(0) && t.size(1) == q.size(1) && t.size(2) == rows[i] &&
               t.size(3) == q.size(3) && t.scalar_type() == q.scalar_type() && t.device() == q.device() &&
               t.stride(3) == 1,
           "out tensors must match q's dtype and device, shaped like (dq, dk, dv), last dimension contiguous");
    }
    dq = (*out)[0], dk = (*out)[1], dv = (*out)[2];
  } else {
    if (need_dq) dq = at::empty(q.sizes(), q.options());
    if (need_dk) dk = at::empty({q.size(0), q.size(1), M, q.size(3)}, q.options());
    dv = at::empty({q.size(0), q.size(1), M, q.size(3)}, q.options());
  }
  const auto p = problem(q, k, scale, causal);
  const auto tq = view(q), tk = view(k), tv = view(v), to = view(o), tdo = view(dout), tdq = view(dq), tdk = view(dk),
             tdv = view(dv);
  check_rc(theria_sdpa_bwd(&p, &tq, &tk, &tv, &to, o_f32 ? 1 : 0, &tdo, fptr(lse),
                           fptr(delta), &tdq, &tdk, &tdv, stream_of(q)),
           "theria_sdpa_bwd");
  return py::make_tuple(dq ? py::cast(*dq) : py::none(), dk ? py::cast(*dk) : py::none(), dv, delta);
}

at::Tensor jvp(at::Tensor q, at::Tensor k, at::Tensor v, OptT o, const at::Tensor& lse_in, const OptT& tq_in,
               const OptT& tk_in, const OptT& tv_in, double scale, bool causal, bool normalize) {
  q = rowmajor(q), k = rowmajor(k), v = rowmajor(v);
  kv_shapes(q, k, v);
  const int64_t T = q.size(2), M = k.size(2);
  const auto tq = like_rows(tq_in, q, T, "tq must have shape (B,H,T,D)");
  const auto tk = like_rows(tk_in, q, M, "tk must have shape (B,H,M,D)");
  const auto tv = like_rows(tv_in, q, M, "tv must have shape (B,H,M,D)");
  if (o) {  // a float32 O of a low-precision op is rebuilt at full precision inside the kernel instead
    if (o->scalar_type() != q.scalar_type())
      o = std::nullopt;
    else
      o = like_rows(*o, q, T, "o must have shape (B,H,T,D)");
  }
  const auto lse = rowstat(lse_in, q, "lse must be a float32 (B,H,T) tensor on q's device");
  const c10::hip::HIPGuard guard(q.get_device());
  const auto out = at::empty(q.sizes(), q.options());
  const auto p = problem(q, k, scale, causal);
  const auto vq = view(q), vk = view(k), vv = view(v), vo = view(o), vtq = view(tq), vtk = view(tk), vtv = view(tv),
             vout = view(out);
  check_rc(theria_sdpa_jvp(&p, &vq, &vk, &vv, &vo, fptr(lse), &vtq, &vtk, &vtv, &vout,
                           normalize ? 1 : 0, stream_of(q)),
           "theria_sdpa_jvp");
  return out;
}

// (G_Q, G_K, G_V, G_dO) as _ops.bwd_bwd; delta is not read by the library and may be None.
py::tuple bwd_bwd(at::Tensor q, at::Tensor k, at::Tensor v, OptT o, const at::Tensor& dout_in,
                  const at::Tensor& lse_in, const OptT& gq_in, const OptT& gk_in, const OptT& gv_in, double scale,
                  bool causal, bool noalloc, const std::optional<std::vector<at::Tensor>>& out) {
  q = rowmajor(q), k = rowmajor(k), v = rowmajor(v);
  kv_shapes(q, k, v);
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), M = k.size(2), D = q.size(3);
  const auto dout = like_rows(dout_in, q, T, "dout must have shape (B,H,T,D)");
  const auto gq = like_rows(gq_in, q, T, "gq must have shape (B,H,T,D)");
  const auto gk = like_rows(gk_in, q, M, "gk must have shape (B,H,M,D)");
  const auto gv = like_rows(gv_in, q, M, "gv must have shape (B,H,M,D)");
  if (o) {
    if (o->scalar_type() != q.scalar_type())
      o = std::nullopt;
    else
      o = like_rows(*o, q, T, "o must have shape (B,H,T,D)");
  }
  const auto lse = rowstat(lse_in, q, "lse must be a float32 (B,H,T) tensor on q's device");
  const c10::hip::HIPGuard guard(q.get_device());
  at::Tensor oq, ok, ov;
  if (out) {
    need(out->size() == 3, "out must hold (out_gq, out_gk, out_gv)");
    const int64_t rows[3] = {T, M, M};
    for (int i = 0; i < 3; ++i) {
      const auto& t = (*out)[i];
      need(t.dim() == 4 && t.size(0) == B && t.size(1) == H && t.size(2) == rows[i] && t.size(3) == D &&
               t.scalar_type() == q.scalar_type() && t.device() == q.device() && t.stride(3) == 1,
           "out tensors must match q's dtype and device, shaped like (gq, gk, gv), last dimension contiguous");
    }
    oq = (*out)[0], ok = (*out)[1], ov = (*out)[2];
  } else {
    oq = at::empty(q.sizes(), q.options());
    ok = at::empty({B, H, M, D}, q.options());
    ov = at::empty({B, H, M, D}, q.options());
  }
  const auto odo = at::empty(q.sizes(), q.options());
  const auto p = problem(q, k, scale, causal);
  const auto vq = view(q), vk = view(k), vv = view(v), vo = view(o), vdo = view(dout), vgq = view(gq), vgk = view(gk),
             vgv = view(gv), voq = view(oq), vok = view(ok), vov = view(ov), vodo = view(odo);
  int rc;
  if (noalloc) {
    rc = theria_sdpa_bwd_bwd_noalloc(&p, &vq, &vk, &vv, &vo, &vdo, fptr(lse), nullptr, &vgq, &vgk, &vgv,
                                     &voq, &vok, &vov, &vodo, stream_of(q));
    check_rc(rc, "theria_sdpa_bwd_bwd_noalloc");
  } else {
    const auto ws = at::empty({5 * B * H * T}, q.options().dtype(at::kFloat));
    rc = theria_sdpa_bwd_bwd(&p, &vq, &vk, &vv, &vo, &vdo, fptr(lse), nullptr, &vgq, &vgk, &vgv, &voq,
                             &vok, &vov, &vodo, fptr(ws), stream_of(q));
    check_rc(rc, "theria_sdpa_bwd_bwd");
  }
  return py::make_tuple(oq, ok, ov, odo);
}

// ---- token-side operators: matrices (rows, width), whose leading dimensions are flattened -------------------------

// A tensor's rows of `width` as a matrix; a copy only where no view with a contiguous last dimension exists.
at::Tensor rows_of(const at::Tensor& t_in, int64_t width) {
  at::Tensor t = plain(t_in);
  if (t.dim() != 2) t = t.reshape({t.numel() / width, width});
  if (width > 1 && t.stride(1) != 1) t = t.contiguous();
  return t;
}
at::Tensor rows_of(const at::Tensor& t, const at::Tensor& like, const char* msg) {
  need(t.sizes() == like.sizes() && t.device() == like.device(), msg);
  return rows_of(t.scalar_type() == like.scalar_type() ? t : t.to(like.scalar_type()), like.size(-1));
}
OptT rows_of(const OptT& t, const at::Tensor& like, const char* msg) {
  if (!t) return std::nullopt;
  return rows_of(*t, like, msg);
}
theria_rows_t rows_view(const at::Tensor& t) { return {t.data_ptr(), t.stride(0)}; }
theria_rows_t rows_view(const OptT& t) { return t ? rows_view(*t) : theria_rows_t{nullptr, 0}; }
void* ptr(const OptT& t) { return t ? plain(*t).data_ptr() : nullptr; }
OptT flat(const OptT& t) {
  if (!t) return std::nullopt;
  return plain(*t).contiguous();
}
py::object given(const OptT& t) { return t ? py::cast(*t) : py::none(); }

theria_layer_norm_problem_t norm_problem(const at::Tensor& x, at::ScalarType param, double eps) {
  return {dtype_code(x.scalar_type()), dtype_code(param), (int32_t)x.size(1), (float)eps, x.size(0)};
}

py::tuple layer_norm_fwd(const at::Tensor& x_in, const OptT& weight_in, const OptT& bias_in, double eps) {
  const int64_t width = x_in.size(-1);
  const at::Tensor x = rows_of(x_in, width);
  const OptT weight = flat(weight_in), bias = flat(bias_in);
  const c10::hip::HIPGuard guard(x.get_device());
  const auto y = at::empty({x.size(0), width}, x.options());
  const auto mean = at::empty({x.size(0)}, x.options().dtype(at::kFloat)), rstd = at::empty_like(mean);
  const auto p = norm_problem(x, weight ? weight->scalar_type() : bias ? bias->scalar_type() : x.scalar_type(), eps);
  const auto vx = rows_view(x), vy = rows_view(y);
  check_rc(theria_layer_norm_fwd(&p, &vx, ptr(weight), ptr(bias), &vy, fptr(mean), fptr(rstd), stream_of(x)),
           "theria_layer_norm_fwd");
  return py::make_tuple(y.view(x_in.sizes()), mean, rstd);
}

py::tuple layer_norm_bwd(const at::Tensor& x_in, const OptT& weight_in, const at::Tensor& dout_in, const at::Tensor& mean,
                         const at::Tensor& rstd, double eps, bool need_dx, bool need_dw, bool need_db, at::ScalarType param) {
  const int64_t width = x_in.size(-1);
  const at::Tensor dout = rows_of(dout_in, x_in, "the gradient must have the shape of the input");
  const at::Tensor x = rows_of(x_in, width);
  const OptT weight = flat(weight_in);
  const c10::hip::HIPGuard guard(x.get_device());
  OptT dx, dw, db, ws;
  if (need_dx) dx = at::empty({x.size(0), width}, x.options());
  const auto po = x.options().dtype(param);
  const bool none = x.size(0) == 0;
  if (need_dw) dw = none ? at::zeros({width}, po) : at::empty({width}, po);
  if (need_db) db = none ? at::zeros({width}, po) : at::empty({width}, po);
  if (!none) {
    const auto p = norm_problem(x, param, eps);
    if (need_dw || need_db) ws = at::empty({theria_layer_norm_ws_floats(&p)}, x.options().dtype(at::kFloat));
    const auto vx = rows_view(x), vg = rows_view(dout), vdx = rows_view(dx);
    check_rc(theria_layer_norm_bwd(&p, &vx, ptr(weight), &vg, fptr(mean), fptr(rstd), &vdx, ptr(dw), ptr(db), fptr(ws), stream_of(x)),
             "theria_layer_norm_bwd");
  }
  if (dx) dx = dx->view(x_in.sizes());
  return py::make_tuple(given(dx), given(dw), given(db));
}

py::tuple layer_norm_bwd_bwd(const at::Tensor& x_in, const OptT& weight_in, const at::Tensor& dout_in, const at::Tensor& mean,
                             const at::Tensor& rstd, double eps, const OptT& gdx_in, const OptT& gdw_in, const OptT& gdb_in,
                             bool need_gx, bool need_gw, bool need_gdout, at::ScalarType param) {
  const int64_t width = x_in.size(-1);
  const at::Tensor dout = rows_of(dout_in, x_in, "the gradient must have the shape of the input");
  const OptT gdx = rows_of(gdx_in, x_in, "a cotangent must have the shape of the input");
  const at::Tensor x = rows_of(x_in, width);
  auto param_like = [&](const OptT& t) -> OptT {
    if (!t) return std::nullopt;
    need(t->numel() == width && t->device() == x.device(), "a cotangent must have the shape of its parameter");
    return flat(t->scalar_type() == param ? *t : t->to(param));
  };
  const OptT weight = flat(weight_in), gdw = param_like(gdw_in), gdb = param_like(gdb_in);
  const c10::hip::HIPGuard guard(x.get_device());
  OptT gx, gw, gg, ws;
  const bool none = x.size(0) == 0;
  if (need_gx) gx = at::empty({x.size(0), width}, x.options());
  if (need_gdout) gg = at::empty({x.size(0), width}, x.options());
  if (need_gw) gw = none ? at::zeros({width}, x.options().dtype(param)) : at::empty({width}, x.options().dtype(param));
  if (!none) {
    const auto p = norm_problem(x, param, eps);
    if (need_gw) ws = at::empty({theria_layer_norm_ws_floats(&p)}, x.options().dtype(at::kFloat));
    const auto vx = rows_view(x), vg = rows_view(dout), vu = rows_view(gdx), vgx = rows_view(gx), vgg = rows_view(gg);
    check_rc(theria_layer_norm_bwd_bwd(&p, &vx, ptr(weight), &vg, fptr(mean), fptr(rstd), &vu, ptr(gdw), ptr(gdb), &vgx, ptr(gw),
                                       &vgg, fptr(ws), stream_of(x)),
             "theria_layer_norm_bwd_bwd");
  }
  if (gx) gx = gx->view(x_in.sizes());
  if (gg) gg = gg->view(x_in.sizes());
  return py::make_tuple(given(gx), given(gw), given(gg));
}

at::Tensor embedding_fwd(const at::Tensor& ids_in, const at::Tensor& table_in, double scale, int64_t padding, bool zero_padding) {
  const int64_t width = table_in.size(1);
  const at::Tensor table = rows_of(table_in, width), ids = plain(ids_in).contiguous();
  const c10::hip::HIPGuard guard(table.get_device());
  const auto out = at::empty({ids.numel(), width}, table.options());
  const theria_embedding_problem_t p{dtype_code(table.scalar_type()), ids.scalar_type() == at::kLong, (int32_t)width,
                                     (float)scale, ids.numel(), table.size(0), padding};
  const auto vt = rows_view(table), vo = rows_view(out);
  check_rc(theria_embedding_fwd(&p, ids.data_ptr(), &vt, zero_padding, &vo, stream_of(table)), "theria_embedding_fwd");
  auto sizes = ids_in.sizes().vec();
  sizes.push_back(width);
  return out.view(sizes);
}

at::Tensor embedding_bwd(const at::Tensor& ids_in, const at::Tensor& dout_in, int64_t classes, double scale, int64_t padding) {
  const int64_t width = dout_in.size(-1);
  const at::Tensor ids = plain(ids_in).contiguous(), dout = rows_of(dout_in, width);
  need(dout.size(0) == ids.numel() && dout.device() == ids.device(), "the gradient must have one row for each id");
  const c10::hip::HIPGuard guard(dout.get_device());
  const auto out = at::empty({classes, width}, dout.options());
  const theria_embedding_problem_t p{dtype_code(dout.scalar_type()), ids.scalar_type() == at::kLong, (int32_t)width,
                                     (float)scale, ids.numel(), classes, padding};
  const auto ws = at::empty({theria_embedding_ws_bytes(&p)}, dout.options().dtype(at::kByte));
  const auto vg = rows_view(dout), vo = rows_view(out);
  check_rc(theria_embedding_bwd(&p, ids.data_ptr(), &vg, &vo, ws.data_ptr(), stream_of(dout)), "theria_embedding_bwd");
  return out;
}

theria_linear_ce_problem_t ce_problem(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& target, int64_t ignore, int reduction) {
  return {dtype_code(x.scalar_type()), target.scalar_type() == at::kLong, reduction, (int32_t)x.size(1), x.size(0), weight.size(0), ignore};
}

// A 256-byte-aligned workspace: torch's allocations are.
at::Tensor ce_workspace(const theria_linear_ce_problem_t& p, const theria_rows_t& w, const at::Tensor& x, bool backward, bool dx, bool dw, bool db) {
  return at::empty({theria_linear_ce_ws_bytes(&p, &w, backward, dx, dw, db)}, x.options().dtype(at::kByte));
}

py::tuple linear_ce_fwd(const at::Tensor& x_in, const at::Tensor& weight_in, const OptT& bias_in, const at::Tensor& target_in,
                        int64_t ignore, int reduction) {
  const int64_t width = x_in.size(-1);
  const at::Tensor x = rows_of(x_in, width), weight = rows_of(weight_in, width), target = plain(target_in).contiguous();
  const OptT bias = flat(bias_in);
  const c10::hip::HIPGuard guard(x.get_device());
  const auto f = x.options().dtype(at::kFloat);
  const auto loss = reduction == THERIA_REDUCE_NONE ? at::empty({x.size(0)}, f) : at::empty({}, f);
  const auto stats = at::empty({2, x.size(0)}, f);
  const auto p = ce_problem(x, weight, target, ignore, reduction);
  const auto vx = rows_view(x), vw = rows_view(weight);
  const auto ws = ce_workspace(p, vw, x, false, false, false, false);
  check_rc(theria_linear_ce_fwd(&p, &vx, &vw, ptr(bias), target.data_ptr(), fptr(loss), fptr(stats), ws.data_ptr(), stream_of(x)),
           "theria_linear_ce_fwd");
  return py::make_tuple(reduction == THERIA_REDUCE_NONE ? loss.view(target_in.sizes()) : loss, stats);
}

py::tuple linear_ce_bwd(const at::Tensor& x_in, const at::Tensor& weight_in, const OptT& bias_in, const at::Tensor& target_in,
                        const at::Tensor& stats, const at::Tensor& dloss_in, int64_t ignore, int reduction, bool need_dx, bool need_dw,
                        bool need_db) {
  const int64_t width = x_in.size(-1);
  const at::Tensor x = rows_of(x_in, width), weight = rows_of(weight_in, width), target = plain(target_in).contiguous();
  const OptT bias = flat(bias_in);
  const at::Tensor dloss = plain(dloss_in).to(at::kFloat).contiguous();
  need(dloss.numel() == (reduction == THERIA_REDUCE_NONE ? x.size(0) : 1) && dloss.device() == x.device(),
       "the loss's gradient must have the shape of the loss");
  const c10::hip::HIPGuard guard(x.get_device());
  OptT dx, dw, db;
  if (need_dx) dx = at::empty({x.size(0), width}, x.options());
  if (need_dw) dw = at::empty({weight.size(0), width}, x.options());
  if (need_db) db = at::empty({weight.size(0)}, x.options());
  const auto p = ce_problem(x, weight, target, ignore, reduction);
  const auto vx = rows_view(x), vw = rows_view(weight), vdx = rows_view(dx), vdw = rows_view(dw);
  const auto ws = ce_workspace(p, vw, x, true, need_dx, need_dw, need_db);
  check_rc(theria_linear_ce_bwd(&p, &vx, &vw, ptr(bias), target.data_ptr(), fptr(stats), fptr(dloss), &vdx, &vdw, ptr(db), ws.data_ptr(),
                                stream_of(x)),
           "theria_linear_ce_bwd");
  if (dx) dx = dx->view(x_in.sizes());
  return py::make_tuple(given(dx), given(dw), given(db));
}

}  // namespace

PYBIND11_MODULE(_theria_host, m) {
  m.doc() = "torch-tensor binding of the hot C ABI entry points of libtheria_sdpa.so";
  m.def("abi_version", &theria_abi_version);
  m.def("fwd", &fwd, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("scale"), py::arg("causal"),
        py::arg("out_fp32"), py::arg("stats"));
  m.def("bwd", &bwd, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("o"), py::arg("lse"), py::arg("dout"),
        py::arg("scale"), py::arg("causal"), py::arg("need_dq"), py::arg("need_dk"), py::arg("out"));
  m.def("jvp", &jvp, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("o"), py::arg("lse"), py::arg("tq"),
        py::arg("tk"), py::arg("tv"), py::arg("scale"), py::arg("causal"), py::arg("normalize"));
  m.def("bwd_bwd", &bwd_bwd, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("o"), py::arg("dout"),
        py::arg("lse"), py::arg("gq"), py::arg("gk"), py::arg("gv"), py::arg("scale"), py::arg("causal"),
        py::arg("noalloc"), py::arg("out"));
  m.def("layer_norm_fwd", &layer_norm_fwd);
  m.def("layer_norm_bwd", &layer_norm_bwd);
  m.def("layer_norm_bwd_bwd", &layer_norm_bwd_bwd);
  m.def("embedding_fwd", &embedding_fwd);
  m.def("embedding_bwd", &embedding_bwd);
  m.def("linear_ce_fwd", &linear_ce_fwd);
  m.def("linear_ce_bwd", &linear_ce_bwd);
}
