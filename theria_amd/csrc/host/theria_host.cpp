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

#include <cmath>
#include <functional>
#include <initializer_list>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

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

// ---- token-side operators -------------------------------------------------------------------------------------------
//
// Matrices are (rows, width) with their leading dimensions flattened. The autograd Functions are C++ too: a training step
// of a small model is bound by the host's time per operator, and a Python Function costs several times a kernel (argument
// packing, and the interpreter lock taken again by the engine's thread): forward and backward of a (1600, 64) layer norm
// took 85 us with Python Functions. An engine thread does not hold the interpreter lock, so nothing here touches
// Python: contract violations are C++ exceptions, translated to AssertionError where the call came from Python.

struct ContractError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
// The message is only put together where it is thrown: the strings of one operator's checks cost as much as its launch.
#define THERIA_MUST(ok, msg) \
  do {                       \
    if (!(ok)) throw ContractError(msg); \
  } while (0)
void token_rc(int rc, const char* what) {
  if (rc == THERIA_OK) return;
  const std::string msg = std::string(what) + ": " + theria_last_error();
  if (rc == THERIA_ERR_CONTRACT) throw ContractError(msg);
  throw std::runtime_error(msg);
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using at::Tensor;

constexpr int64_t kMaxNormWidth = 16384, kMaxRowWidth = 1 << 20, kMaxRows = (int64_t(1) << 31) - 64;

int32_t token_dtype(at::ScalarType st) { return st == at::kFloat ? THERIA_DTYPE_F32 : st == at::kHalf ? THERIA_DTYPE_F16 : THERIA_DTYPE_BF16; }

std::string shape_text(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}

// A torch.func transform wraps its tensors; the C++ Functions know nothing of that.
void check_plain(const Tensor& t, const char* what) { THERIA_MUST(t.has_storage(), std::string(what) + " does not run under torch.func transforms"); }

// Device, dtype and size contract of the operators' matrices.
void check_matrix(const Tensor& t, const char* name, const char* what) {
  THERIA_MUST(t.defined(), std::string(what) + ": " + name + " must be a tensor");
  THERIA_MUST(t.is_cuda(), std::string(what) + " requires GPU (HIP) tensors; " + name + " is on " + t.device().str());
  check_plain(t, what);
  const auto st = t.scalar_type();
  THERIA_MUST(st == at::kFloat || st == at::kHalf || st == at::kBFloat16, std::string("Unsupported dtype for ") + name + ": " + c10::toString(st));
  THERIA_MUST(t.dim() == 0 || t.size(-1) == 0 || t.numel() / t.size(-1) <= kMaxRows, std::string(what) + ": " + name + " has more rows than 32-bit indexes reach");
}
// Ids or targets.
void check_indexes(const Tensor& t, const char* name, const Tensor& like, const char* what) {
  THERIA_MUST(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, std::string(what) + ": " + name + " must be an int32 or int64 tensor");
  THERIA_MUST(t.device() == like.device(), std::string(what) + ": " + name + " must be on " + like.device().str() + ", got " + t.device().str());
  check_plain(t, what);
  THERIA_MUST(t.numel() <= kMaxRows, std::string(what) + ": " + name + " has more elements than 32-bit indexes reach");
}

// A tensor's rows of `width` as a matrix; a copy only where no view with a contiguous last dimension exists, or where the
// view is one of negated values (the imaginary part of a conjugate).
Tensor rows_of(const Tensor& t_in, int64_t width) {
  Tensor t = t_in.resolve_neg();
  if (t.dim() != 2) t = t.reshape({t.numel() / width, width});
  if (width > 1 && t.stride(1) != 1) t = t.contiguous();
  return t;
}
// A gradient or cotangent in the shape and type of `like`; undefined stays undefined.
Tensor rows_like(const Tensor& t, const Tensor& like, const char* what) {
  if (!t.defined()) return t;
  THERIA_MUST(t.sizes() == like.sizes() && t.device() == like.device(), std::string(what) + ": a gradient must have the shape of its input");
  return rows_of(t.scalar_type() == like.scalar_type() ? t : t.to(like.scalar_type()), like.size(-1));
}
Tensor flat(const Tensor& t) { return t.defined() ? t.resolve_neg().contiguous() : t; }
theria_rows_t rows_view(const Tensor& t) { return t.defined() ? theria_rows_t{t.data_ptr(), t.stride(0)} : theria_rows_t{nullptr, 0}; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* floats(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

// The gradients of `outs` (with cotangents `cots`) with respect to aliases of `prim` that require them, by autograd through
// `map`: the derivatives that no kernel covers. Aliases, so that each result is a partial derivative. keep: with a graph of
// their own (through the originals); else the inputs are cut off first.
template <class Map>
variable_list through_map(const variable_list& prim, const std::vector<bool>& want, const variable_list& cots, bool keep, const Map& map) {
  const at::AutoGradMode grad(true);
  variable_list alias, wrt, outs, gs;
  for (size_t i = 0; i < prim.size(); ++i) {
    alias.push_back(!want[i] || !prim[i].defined() ? prim[i] : keep ? prim[i].view_as(prim[i]) : prim[i].detach().requires_grad_(true));
    if (want[i] && prim[i].defined()) wrt.push_back(alias.back());
  }
  const variable_list all = map(alias);
  for (size_t i = 0; i < all.size(); ++i)
    if (cots[i].defined() && all[i].requires_grad()) outs.push_back(all[i]), gs.push_back(cots[i].to(all[i].scalar_type()));
  variable_list result(prim.size());
  if (outs.empty() || wrt.empty()) return result;
  const variable_list got = torch::autograd::grad(outs, wrt, gs, /*retain_graph=*/keep, /*create_graph=*/keep, /*allow_unused=*/true);
  size_t k = 0;
  for (size_t i = 0; i < prim.size(); ++i)
    if (want[i] && prim[i].defined()) result[i] = got[k++];
  return result;
}

// A Function's outputs are the gradients that are wanted, without the others: packed from, and its cotangents unpacked to,
// a list with a place for each.
variable_list packed(const variable_list& all) {
  variable_list some;
  for (const Tensor& t : all)
    if (t.defined()) some.push_back(t);
  return some;
}
variable_list unpacked(const variable_list& some, const std::vector<bool>& want) {
  variable_list all(want.size());
  size_t k = 0;
  for (size_t i = 0; i < want.size(); ++i)
    if (want[i]) all[i] = some[k++];
  return all;
}

// A Function's inputs are all defined: an absent parameter goes in as an empty tensor and comes out undefined again.
Tensor or_empty(const Tensor& t, const Tensor& like) { return t.defined() ? t : at::empty({0}, like.options()); }
Tensor or_absent(const Tensor& t) { return t.numel() ? t : Tensor(); }

// Whether a call is outside autograd altogether, so that it runs without a Function (0.7 us of its 4 to 6). A forward-mode
// tangent is not: the Function refuses it.
bool outside_autograd(std::initializer_list<std::reference_wrapper<const Tensor>> inputs) {
  for (const Tensor& t : inputs)
    if (t.defined() && ((at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined())) return false;
  return true;
}

std::vector<bool> needed(AutogradContext* ctx) {
  const auto list = ctx->saved_data["need"].toBoolList();
  return std::vector<bool>(list.begin(), list.end());
}

// ---- layer norm
theria_layer_norm_problem_t norm_problem(const Tensor& x, at::ScalarType param, double eps) {
  return {token_dtype(x.scalar_type()), token_dtype(param), (int32_t)x.size(1), (float)eps, x.size(0)};
}

variable_list norm_bwd(const Tensor& x_in, const Tensor& weight_in, const Tensor& dy_in, const Tensor& stats, double eps,
                       at::ScalarType param, bool need_dx, bool need_dw, bool need_db) {
  const int64_t width = x_in.size(-1);
  const Tensor dy = rows_like(dy_in, x_in, "hip_layer_norm"), x = rows_of(x_in, width), weight = flat(weight_in);
  const c10::hip::HIPGuard guard(x.get_device());
  Tensor dx, dw, db, ws;
  if (need_dx) dx = at::empty(x_in.sizes(), x.options());
  const auto po = x.options().dtype(param);
  const bool none = x.size(0) == 0;
  if (need_dw) dw = none ? at::zeros({width}, po) : at::empty({width}, po);
  if (need_db) db = none ? at::zeros({width}, po) : at::empty({width}, po);
  if (!none) {
    const auto p = norm_problem(x, param, eps);
    if (need_dw || need_db) ws = at::empty({theria_layer_norm_ws_floats(&p)}, x.options().dtype(at::kFloat));
    const auto vx = rows_view(x), vg = rows_view(dy);
    const theria_rows_t vdx{ptr(dx), width};
    token_rc(theria_layer_norm_bwd(&p, &vx, ptr(weight), &vg, floats(stats), floats(stats) + x.size(0), &vdx, ptr(dw), ptr(db), floats(ws), stream_of(x)),
             "theria_layer_norm_bwd");
  }
  return {dx, dw, db};
}

variable_list norm_bwd_bwd(const Tensor& x_in, const Tensor& weight_in, const Tensor& dy_in, const Tensor& stats, double eps,
                           at::ScalarType param, const Tensor& u_in, const Tensor& a_in, const Tensor& c_in, bool need_gx, bool need_gw,
                           bool need_gdy) {
  const int64_t width = x_in.size(-1);
  const Tensor dy = rows_like(dy_in, x_in, "hip_layer_norm"), u = rows_like(u_in, x_in, "hip_layer_norm"), x = rows_of(x_in, width),
               weight = flat(weight_in);
  auto param_like = [&](const Tensor& t) {
    if (!t.defined()) return t;
    THERIA_MUST(t.numel() == width && t.device() == x.device(), "hip_layer_norm: a cotangent must have the shape of its parameter");
    return flat(t.scalar_type() == param ? t : t.to(param));
  };
  const Tensor a = param_like(a_in), c = param_like(c_in);
  const c10::hip::HIPGuard guard(x.get_device());
  Tensor gx, gw, gdy, ws;
  const bool none = x.size(0) == 0;
  const auto po = x.options().dtype(param);
  if (need_gx) gx = at::empty(x_in.sizes(), x.options());
  if (need_gdy) gdy = at::empty(x_in.sizes(), x.options());
  if (need_gw) gw = none ? at::zeros({width}, po) : at::empty({width}, po);
  if (!none) {
    const auto p = norm_problem(x, param, eps);
    if (need_gw) ws = at::empty({theria_layer_norm_ws_floats(&p)}, x.options().dtype(at::kFloat));
    const auto vx = rows_view(x), vg = rows_view(dy), vu = rows_view(u);
    const theria_rows_t vgx{ptr(gx), width}, vgdy{ptr(gdy), width};
    token_rc(theria_layer_norm_bwd_bwd(&p, &vx, ptr(weight), &vg, floats(stats), floats(stats) + x.size(0), &vu, ptr(a), ptr(c), &vgx, ptr(gw), &vgdy,
                                       floats(ws), stream_of(x)),
             "theria_layer_norm_bwd_bwd");
  }
  if (gdy.defined() && dy_in.scalar_type() != gdy.scalar_type()) gdy = gdy.to(dy_in.scalar_type());
  return {gx, gw, gdy};
}

// (dx, dweight, dbias) as differentiable torch operations, in float32 or wider: orders three and higher only.
variable_list norm_map(const variable_list& in, double eps) {
  const Tensor &x_in = in[0], &weight = in[1], &dy_in = in[2];
  const int64_t width = x_in.size(-1);
  const auto ct = at::promote_types(x_in.scalar_type(), at::kFloat);
  const Tensor x = x_in.to(ct).reshape({-1, width}), dy = dy_in.to(ct).reshape({-1, width});
  const Tensor xc = x - x.mean(1, true);
  const Tensor rstd = ((xc * xc).mean(1, true) + eps).rsqrt(), xh = xc * rstd;
  const Tensor gw = weight.defined() ? dy * weight.to(ct) : dy;
  const Tensor dx = rstd * (gw - gw.mean(1, true) - xh * (gw * xh).mean(1, true));
  return {dx.reshape(x_in.sizes()).to(x_in.scalar_type()), (dy * xh).sum(0), dy.sum(0)};
}

// (x, weight, dy, stats) -> (dx, dweight, dbias). The statistics are functions of x, whose part in the derivative the
// double backward's kernel includes.
struct NormBackwardFn : torch::autograd::Function<NormBackwardFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight_in, const Tensor& dy, const Tensor& stats,
                               double eps, int64_t param, bool need_dx, bool need_dw, bool need_db) {
    const Tensor weight = or_absent(weight_in);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, weight_in, dy, stats});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["param"] = param;
    ctx->saved_data["need"] = std::vector<bool>{need_dx, need_dw, need_db};
    return packed(norm_bwd(x, weight, dy, stats, eps, (at::ScalarType)param, need_dx, need_dw, need_db));
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& some) {
    variable_list out(9);
    const variable_list g = unpacked(some, needed(ctx));
    if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], weight = or_absent(saved[1]), &dy = saved[2];
    const double eps = ctx->saved_data["eps"].toDouble();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), ny = ctx->needs_input_grad(2);
    const bool keep = at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(dy) || wants(g[0]) || wants(g[1]) || wants(g[2]));
    const variable_list r = keep ? through_map({x, weight, dy}, {nx, nw, ny}, {g[0], g[1], g[2]}, true, [&](const variable_list& in) { return norm_map(in, eps); })
                                 : norm_bwd_bwd(x, weight, dy, saved[3], eps, (at::ScalarType)ctx->saved_data["param"].toInt(), g[0], g[1], g[2], nx, nw, ny);
    out[0] = r[0], out[1] = r[1], out[2] = r[2];
    return out;
  }
};

// y and the statistics (mean, rstd) of each row.
std::pair<Tensor, Tensor> norm_fwd(const Tensor& x_in, const Tensor& weight_in, const Tensor& bias_in, double eps, at::ScalarType param) {
  const int64_t width = x_in.size(-1);
  const Tensor x = rows_of(x_in, width), weight = flat(weight_in), bias = flat(bias_in);
  const c10::hip::HIPGuard guard(x.get_device());
  const Tensor y = at::empty(x_in.sizes(), x.options()), stats = at::empty({2, x.size(0)}, x.options().dtype(at::kFloat));
  const auto p = norm_problem(x, param, eps);
  const auto vx = rows_view(x);
  const theria_rows_t vy{ptr(y), width};
  token_rc(theria_layer_norm_fwd(&p, &vx, ptr(weight), ptr(bias), &vy, floats(stats), floats(stats) + x.size(0), stream_of(x)), "theria_layer_norm_fwd");
  return {y, stats};
}

struct NormFn : torch::autograd::Function<NormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& weight_in, const Tensor& bias_in, double eps, int64_t param) {
    const auto [y, stats] = norm_fwd(x_in, or_absent(weight_in), or_absent(bias_in), eps, (at::ScalarType)param);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x_in, weight_in, stats});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["param"] = param;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    variable_list out(5);
    if (!g[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], weight = or_absent(saved[1]);
    const double eps = ctx->saved_data["eps"].toDouble();
    const int64_t param = ctx->saved_data["param"].toInt();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nb = ctx->needs_input_grad(2);
    const variable_list r = at::GradMode::is_enabled()
                                ? unpacked(NormBackwardFn::apply(x, saved[1], g[0], saved[2], eps, param, nx, nw, nb), {nx, nw, nb})
                                : norm_bwd(x, weight, g[0], saved[2], eps, (at::ScalarType)param, nx, nw, nb);
    out[0] = r[0], out[1] = r[1], out[2] = r[2];
    return out;
  }
};

Tensor layer_norm(const Tensor& x, const OptT& weight_in, const OptT& bias_in, double eps) {
  const char* what = "hip_layer_norm";
  const Tensor weight = weight_in.value_or(Tensor()), bias = bias_in.value_or(Tensor());
  check_matrix(x, "x", what);
  THERIA_MUST(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= kMaxNormWidth,
       std::string(what) + " supports rows of 1 to " + std::to_string(kMaxNormWidth) + " elements, got shape " + shape_text(x));
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>("weight", weight), std::pair<const char*, const Tensor&>("bias", bias)}) {
    if (!t.defined()) continue;
    check_plain(t, what);
    THERIA_MUST(t.dim() == 1 && t.size(0) == x.size(-1), std::string(name) + " must have shape (" + std::to_string(x.size(-1)) + ",), got " + shape_text(t));
    THERIA_MUST((t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat) && t.device() == x.device(),
         std::string(what) + ": " + name + " must be on " + x.device().str() + " in " + c10::toString(x.scalar_type()) + " or float32, got " +
             c10::toString(t.scalar_type()) + " on " + t.device().str());
  }
  THERIA_MUST(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(), std::string(what) + ": weight and bias must have one dtype");
  THERIA_MUST(eps >= 0 && std::isfinite(eps), std::string(what) + ": eps must be finite and not negative, got " + std::to_string(eps));
  const auto param = weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type();
  if (outside_autograd({x, weight, bias})) return norm_fwd(x, weight, bias, eps, param).first;
  return NormFn::apply(x, or_empty(weight, x), or_empty(bias, x), eps, (int64_t)param);
}

// ---- embedding: linear in the table, so that the gradient's derivative is a lookup again
theria_embedding_problem_t embed_problem(const Tensor& ids, const Tensor& rows, int64_t classes, double scale, int64_t padding) {
  return {token_dtype(rows.scalar_type()), ids.scalar_type() == at::kLong, (int32_t)rows.size(1), (float)scale, ids.numel(), classes, padding};
}

Tensor embed_bwd(const Tensor& ids_in, const Tensor& dout_in, int64_t classes, double scale, int64_t padding) {
  const int64_t width = dout_in.size(-1);
  const Tensor ids = ids_in.contiguous(), dout = rows_of(dout_in, width);
  THERIA_MUST(dout.size(0) == ids.numel() && dout.device() == ids.device(), "hip_embedding: the gradient must have one row for each id");
  const c10::hip::HIPGuard guard(dout.get_device());
  const Tensor out = at::empty({classes, width}, dout.options());
  const auto p = embed_problem(ids, dout, classes, scale, padding);
  const Tensor ws = at::empty({theria_embedding_ws_bytes(&p)}, dout.options().dtype(at::kByte));
  const auto vg = rows_view(dout), vo = rows_view(out);
  token_rc(theria_embedding_bwd(&p, ids.data_ptr(), &vg, &vo, ws.data_ptr(), stream_of(dout)), "theria_embedding_bwd");
  return out;
}

struct EmbedBackwardFn : torch::autograd::Function<EmbedBackwardFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& dout, const Tensor& ids, int64_t classes, double scale, int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return embed_bwd(ids, dout, classes, scale, padding);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g);
};

Tensor embed_fwd(const Tensor& table_in, const Tensor& ids_in, double scale, int64_t padding, bool zero_padding) {
  const int64_t width = table_in.size(1);
  const Tensor table = rows_of(table_in, width), ids = ids_in.contiguous();
  const c10::hip::HIPGuard guard(table.get_device());
  at::DimVector sizes(ids_in.sizes());
  sizes.push_back(width);
  const Tensor out = at::empty(sizes, table.options());
  const auto p = embed_problem(ids, table, table.size(0), scale, padding);
  const auto vt = rows_view(table);
  const theria_rows_t vo{ptr(out), width};
  token_rc(theria_embedding_fwd(&p, ids.data_ptr(), &vt, zero_padding, &vo, stream_of(table)), "theria_embedding_fwd");
  return out;
}

struct EmbedFn : torch::autograd::Function<EmbedFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& ids_in, double scale, int64_t padding, bool zero_padding) {
    const Tensor out = embed_fwd(table, ids_in, scale, padding, zero_padding);
    ctx->save_for_backward({ids_in});
    ctx->saved_data["classes"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const Tensor ids = ctx->get_saved_variables()[0];
    const int64_t classes = ctx->saved_data["classes"].toInt(), padding = ctx->saved_data["padding"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    variable_list out(5);
    out[0] = at::GradMode::is_enabled() ? EmbedBackwardFn::apply(g[0], ids, classes, scale, padding) : embed_bwd(ids, g[0], classes, scale, padding);
    return out;
  }
};

variable_list EmbedBackwardFn::backward(AutogradContext* ctx, const variable_list& g) {
  variable_list out(5);
  out[0] = EmbedFn::apply(g[0], ctx->get_saved_variables()[0], ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt(), true);
  return out;
}

Tensor embedding(const Tensor& ids, const Tensor& weight, double scale, std::optional<int64_t> padding_idx) {
  const char* what = "hip_embedding";
  check_matrix(weight, "weight", what);
  THERIA_MUST(weight.dim() == 2 && weight.size(1) >= 1 && weight.size(1) <= kMaxRowWidth,
       std::string(what) + ": weight must be (V, D) with 1 <= D <= " + std::to_string(kMaxRowWidth) + ", got shape " + shape_text(weight));
  check_indexes(ids, "ids", weight, what);
  int64_t padding = -1;
  if (padding_idx) {
    padding = *padding_idx < 0 ? *padding_idx + weight.size(0) : *padding_idx;
    THERIA_MUST(padding >= 0 && padding < weight.size(0), std::string(what) + ": padding_idx " + std::to_string(*padding_idx) + " is outside the table of " +
                                                       std::to_string(weight.size(0)) + " rows");
  }
  THERIA_MUST(std::isfinite(scale) && std::isfinite((float)scale), std::string(what) + ": scale must be finite, got " + std::to_string(scale));
  if (outside_autograd({weight})) return embed_fwd(weight, ids, scale, padding, false);
  return EmbedFn::apply(weight, ids, scale, padding, false);
}

// ---- linear cross entropy
theria_linear_ce_problem_t ce_problem(const Tensor& x, const Tensor& weight, const Tensor& target, int64_t ignore, int64_t reduction) {
  return {token_dtype(x.scalar_type()), target.scalar_type() == at::kLong, (int32_t)reduction, (int32_t)x.size(1), x.size(0), weight.size(0), ignore};
}

// A 256-byte-aligned workspace: torch's allocations are.
Tensor ce_workspace(const theria_linear_ce_problem_t& p, const theria_rows_t& w, const Tensor& x, bool backward, bool dx, bool dw, bool db) {
  return at::empty({theria_linear_ce_ws_bytes(&p, &w, backward, dx, dw, db)}, x.options().dtype(at::kByte));
}

variable_list ce_bwd(const Tensor& x_in, const Tensor& weight_in, const Tensor& bias_in, const Tensor& target_in, const Tensor& stats,
                     const Tensor& dloss_in, int64_t ignore, int64_t reduction, bool need_dx, bool need_dw, bool need_db) {
  const int64_t width = x_in.size(-1);
  const Tensor x = rows_of(x_in, width), weight = rows_of(weight_in, width), target = target_in.contiguous(), bias = flat(bias_in);
  const Tensor dloss = dloss_in.to(at::kFloat).resolve_neg().contiguous();
  THERIA_MUST(dloss.numel() == (reduction == THERIA_REDUCE_NONE ? x.size(0) : 1) && dloss.device() == x.device(),
       "hip_linear_cross_entropy: the loss's gradient must have the shape of the loss");
  const c10::hip::HIPGuard guard(x.get_device());
  Tensor dx, dw, db;
  if (need_dx) dx = at::empty(x_in.sizes(), x.options());
  if (need_dw) dw = at::empty({weight.size(0), width}, x.options());
  if (need_db) db = at::empty({weight.size(0)}, x.options());
  const auto p = ce_problem(x, weight, target, ignore, reduction);
  const auto vx = rows_view(x), vw = rows_view(weight), vdw = rows_view(dw);
  const theria_rows_t vdx{ptr(dx), width};
  const Tensor ws = ce_workspace(p, vw, x, true, need_dx, need_dw, need_db);
  token_rc(theria_linear_ce_bwd(&p, &vx, &vw, ptr(bias), target.data_ptr(), floats(stats), floats(dloss), &vdx, &vdw, ptr(db), ws.data_ptr(),
                                stream_of(x)),
           "theria_linear_ce_bwd");
  return {dx, dw, db};
}

// (dx, dweight, dbias) as differentiable torch operations, in float32 or wider, with the logits materialised. in: x, weight,
// bias, the loss's gradient.
variable_list ce_map(const variable_list& in, const Tensor& target, int64_t ignore, int64_t reduction) {
  const Tensor &x = in[0], &weight = in[1], &bias = in[2];
  const auto ct = at::promote_types(x.scalar_type(), at::kFloat);
  const int64_t V = weight.size(0), D = weight.size(1);
  const Tensor t = target.reshape({-1}).to(at::kLong);
  const Tensor kept = t.ne(ignore).logical_and(t.ge(0)).logical_and(t.lt(V));
  const Tensor zero = at::zeros({}, x.options().dtype(ct));
  const Tensor xf = at::where(kept.unsqueeze(1), x.to(ct).reshape({-1, D}), zero), wf = weight.to(ct);
  Tensor z = at::matmul(xf, wf.t());
  if (bias.defined()) z = z + bias.to(ct);
  const Tensor classes = at::arange(V, t.options());
  const Tensor onehot = at::where(kept, t, at::full({}, -1, t.options())).unsqueeze(1).eq(classes).to(ct);
  Tensor up = at::where(kept, in[3].to(ct).reshape({-1}).expand({t.size(0)}), zero);
  if (reduction == THERIA_REDUCE_MEAN) up = up / kept.sum().clamp_min(1).to(ct);
  const Tensor dz = (at::softmax(z, 1) - onehot) * up.unsqueeze(1);
  return {at::matmul(dz, wf).reshape(x.sizes()).to(x.scalar_type()), at::matmul(dz.t(), xf).to(weight.scalar_type()), dz.sum(0)};
}

struct CeBackwardFn : torch::autograd::Function<CeBackwardFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& target,
                               const Tensor& stats, const Tensor& dloss, int64_t ignore, int64_t reduction, bool need_dx, bool need_dw,
                               bool need_db) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, weight, bias, target, dloss});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["need"] = std::vector<bool>{need_dx, need_dw, need_db};
    return packed(ce_bwd(x, weight, or_absent(bias), target, stats, dloss, ignore, reduction, need_dx, need_dw, need_db));
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& some) {
    variable_list out(11);
    const variable_list g = unpacked(some, needed(ctx));
    if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const int64_t ignore = ctx->saved_data["ignore"].toInt(), reduction = ctx->saved_data["reduction"].toInt();
    const std::vector<bool> want{ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2), ctx->needs_input_grad(5)};
    const variable_list r = through_map({saved[0], saved[1], or_absent(saved[2]), saved[4]}, want, {g[0], g[1], g[2]}, at::GradMode::is_enabled(),
                                        [&](const variable_list& in) { return ce_map(in, saved[3], ignore, reduction); });
    out[0] = r[0], out[1] = r[1], out[2] = r[2], out[5] = r[3];
    return out;
  }
};

// The loss, and the rows' statistics for the backward.
std::pair<Tensor, Tensor> ce_fwd(const Tensor& x_in, const Tensor& weight_in, const Tensor& bias_in, const Tensor& target_in, int64_t ignore,
                                 int64_t reduction) {
  const Tensor x = rows_of(x_in, x_in.size(-1)), weight = rows_of(weight_in, weight_in.size(1)), target = target_in.contiguous(), bias = flat(bias_in);
  const c10::hip::HIPGuard guard(x.get_device());
  const auto f = x.options().dtype(at::kFloat);
  const Tensor loss = reduction == THERIA_REDUCE_NONE ? at::empty(target_in.sizes(), f) : at::empty({}, f);
  const Tensor stats = at::empty({2, x.size(0)}, f);
  const auto p = ce_problem(x, weight, target, ignore, reduction);
  const auto vx = rows_view(x), vw = rows_view(weight);
  const Tensor ws = ce_workspace(p, vw, x, false, false, false, false);
  token_rc(theria_linear_ce_fwd(&p, &vx, &vw, ptr(bias), target.data_ptr(), floats(loss), floats(stats), ws.data_ptr(), stream_of(x)),
           "theria_linear_ce_fwd");
  return {loss, stats};
}

struct CeFn : torch::autograd::Function<CeFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& weight_in, const Tensor& bias_in, const Tensor& target_in,
                        int64_t ignore, int64_t reduction) {
    const auto [loss, stats] = ce_fwd(x_in, weight_in, or_absent(bias_in), target_in, ignore, reduction);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x_in, weight_in, bias_in, target_in, stats});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["reduction"] = reduction;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    variable_list out(6);
    if (!g[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const int64_t ignore = ctx->saved_data["ignore"].toInt(), reduction = ctx->saved_data["reduction"].toInt();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nb = ctx->needs_input_grad(2);
    const variable_list r = at::GradMode::is_enabled()
                                ? unpacked(CeBackwardFn::apply(saved[0], saved[1], saved[2], saved[3], saved[4], g[0], ignore, reduction, nx, nw, nb), {nx, nw, nb})
                                : ce_bwd(saved[0], saved[1], or_absent(saved[2]), saved[3], saved[4], g[0], ignore, reduction, nx, nw, nb);
    out[0] = r[0], out[1] = r[1], out[2] = r[2];
    return out;
  }
};

Tensor linear_cross_entropy(const Tensor& x, const Tensor& weight, const Tensor& target, const OptT& bias_in, int64_t ignore, const std::string& reduction) {
  const char* what = "hip_linear_cross_entropy";
  const std::string w = what;
  const Tensor bias = bias_in.value_or(Tensor());
  check_matrix(x, "x", what);
  check_matrix(weight, "weight", what);
  THERIA_MUST(x.dim() >= 1 && weight.dim() == 2 && x.size(-1) == weight.size(1),
       w + ": x must be (..., D) and weight (V, D), got " + shape_text(x) + " and " + shape_text(weight));
  THERIA_MUST(weight.size(0) >= 1 && weight.size(1) >= 1 && weight.size(1) <= kMaxRowWidth,
       w + " supports V >= 1 and 1 <= D <= " + std::to_string(kMaxRowWidth) + ", got weight " + shape_text(weight));
  THERIA_MUST(weight.scalar_type() == x.scalar_type() && weight.device() == x.device(), w + ": weight must match x in dtype and device");
  if (bias.defined()) check_plain(bias, what);
  THERIA_MUST(!bias.defined() || (bias.dim() == 1 && bias.size(0) == weight.size(0) && bias.scalar_type() == x.scalar_type() &&
                           bias.device() == x.device()),
       w + ": bias must be (" + std::to_string(weight.size(0)) + ",) and match x in dtype and device");
  check_indexes(target, "target", x, what);
  THERIA_MUST(target.sizes() == x.sizes().slice(0, x.dim() - 1), w + ": target must have shape " + "x's without its last dimension, got " + shape_text(target) +
                                                              " for x " + shape_text(x));
  THERIA_MUST(reduction == "none" || reduction == "mean" || reduction == "sum", w + ": reduction must be 'none', 'mean' or 'sum', got '" + reduction + "'");
  const int64_t r = reduction == "none" ? THERIA_REDUCE_NONE : reduction == "mean" ? THERIA_REDUCE_MEAN : THERIA_REDUCE_SUM;
  if (outside_autograd({x, weight, bias})) return ce_fwd(x, weight, bias, target, ignore, r).first;
  return CeFn::apply(x, weight, or_empty(bias, x), target, ignore, r);
}

// The differentiable restatements, for tests without a GPU.
py::tuple norm_map_py(const Tensor& x, const OptT& w, const Tensor& dy, double eps) {
  const auto r = norm_map({x, w.value_or(Tensor()), dy}, eps);
  return py::make_tuple(r[0], r[1], r[2]);
}
py::tuple ce_map_py(const Tensor& x, const Tensor& w, const OptT& b, const Tensor& target, const Tensor& dloss, int64_t ignore, int64_t reduction) {
  const auto r = ce_map({x, w, b.value_or(Tensor()), dloss}, target, ignore, reduction);
  return py::make_tuple(r[0], r[1], r[2]);
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
  py::register_exception_translator([](std::exception_ptr e) {
    try {
      if (e) std::rethrow_exception(e);
    } catch (const ContractError& x) {
      PyErr_SetString(PyExc_AssertionError, x.what());
    }
  });
  m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("eps"));
  m.def("embedding", &embedding, py::arg("ids"), py::arg("weight"), py::arg("scale"), py::arg("padding_idx"));
  m.def("linear_cross_entropy", &linear_cross_entropy, py::arg("x"), py::arg("weight"), py::arg("target"), py::arg("bias"),
        py::arg("ignore_index"), py::arg("reduction"));
  m.def("layer_norm_backward_map", &norm_map_py);
  m.def("linear_ce_backward_map", &ce_map_py);
}
