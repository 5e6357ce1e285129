// The parts of operators that run on the host for every call and took longer
// from Python than their kernels do.
//
//   gather   what an optimizer step asks of hundreds of tensors: 512 parameters'
//            and gradients' sizes, types, devices, layouts and addresses take
//            some 250 us one attribute at a time, 10 us here.
//   changed  the versions of what that step has written.
//   linear   the linear layer over the C ABI, and its place in autograd: the
//            engine calls a backward that is written in Python with the
//            interpreter's lock, on a thread of its own.
//   token_logprobs, logits_grad, preference, policy   the losses' outputs,
//            workspaces and calls.
#include <Python.h>

#include <cstring>
#include <string>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include "mhc_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ------------------------------------------------------------- the C ABI --
// Entry points of the library that the process has loaded (bind).
struct Library {
  decltype(&mhc_linear_fwd_workspace_bytes) fwd_bytes;
  decltype(&mhc_linear_fwd) fwd;
  decltype(&mhc_linear_bwd_workspace_bytes) bwd_bytes;
  decltype(&mhc_linear_bwd) bwd;
  decltype(&mhc_token_logprobs) token_logprobs;
  decltype(&mhc_logits_grad) logits_grad;
  decltype(&mhc_preference_loss) preference;
  decltype(&mhc_policy_workspace_bytes) policy_bytes;
  decltype(&mhc_policy_loss) policy;
  decltype(&mhc_last_error) last_error;
} lib = {};

PyObject* mhc_error = nullptr;  // the package's exception for a call that failed (bind)

// As the package's own calls over the C ABI: ValueError for bad arguments, MHCError for
// the rest.  The interpreter's lock may be held or not.
void check(int status, const char* fn) {
  if (status == MHC_OK) return;
  TORCH_CHECK_VALUE(status != MHC_ERR_INVALID, fn, ": ", lib.last_error());
  const std::string text = lib.last_error();  // of this thread
  const pybind11::gil_scoped_acquire locked;
  PyObject* e = PyObject_CallFunction(mhc_error, "sis", fn, status, text.c_str());
  if (e) {
    PyErr_SetObject(mhc_error, e);
    Py_DECREF(e);
  }
  python_error error;
  error.persist();  // it may travel to another thread, from the autograd engine's
  throw error;
}
void* stream_of(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor workspace(size_t bytes, const Tensor& like) {
  if (bytes == 0) return {};
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

// Outputs carry no tangent of forward-mode differentiation: one that came in would be
// taken for 0.
void require_no_tangent(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(),
                              "mhc_b200: no forward-mode differentiation of this operator");
}
// All on x's device, which is a GPU, and without a tangent; undefined ones do not count.
void require_cuda(const Tensor& x, std::initializer_list<const Tensor*> others) {
  TORCH_CHECK(lib.fwd != nullptr, "the library is not loaded");
  const auto one = [&](const Tensor& t) {
    if (!t.defined()) return;
    TORCH_CHECK(t.is_cuda(), "mhc_b200 runs only on CUDA tensors (sm_100a kernels); got a tensor on ",
                t.device(), ".  There is no CPU fallback.");
    TORCH_CHECK_VALUE(t.device() == x.device(), "tensors on different devices: ", x.device(), " and ",
                      t.device());
    require_no_tangent(t);
  };
  one(x);
  for (const Tensor* t : others) one(*t);
}

// A call's arguments.
struct Args {
  const char* fn;
  PyObject* const* v;
  Args(const char* fn_, PyObject* const* v_, Py_ssize_t n, Py_ssize_t want) : fn(fn_), v(v_) {
    TORCH_CHECK_TYPE(n == want, fn, ": ", want, " arguments are expected, got ", n);
  }
  const Tensor& tensor(int i) const {
    TORCH_CHECK_TYPE(THPVariable_Check(v[i]), fn, ": argument ", i, " must be a tensor");
    return THPVariable_Unpack(v[i]);
  }
  Tensor maybe(int i) const { return v[i] == Py_None ? Tensor() : tensor(i); }
  int64_t integer(int i) const {
    const long long k = PyLong_AsLongLong(v[i]);
    if (k == -1 && PyErr_Occurred()) throw python_error();
    return k;
  }
  float number(int i) const {
    const double d = PyFloat_AsDouble(v[i]);
    if (d == -1.0 && PyErr_Occurred()) throw python_error();
    return (float)d;
  }
};
PyObject* tuple_of(std::initializer_list<Tensor> ts) {
  PyObject* out = PyTuple_New((Py_ssize_t)ts.size());
  if (!out) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor& t : ts) {
    PyObject* o = t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None);
    if (!o) {
      Py_DECREF(out);
      throw python_error();
    }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

// ----------------------------------------------------------- linear layer --
// [..., C] taken as rows: in place where the strides allow, else a copy.
struct Rows {
  Tensor t;
  int64_t ld = 0;  // distance between rows
  explicit Rows(const Tensor& x) : t(x) {
    if (!x.defined()) return;
    if (x.is_neg()) t = x.resolve_neg();
    const int64_t c = x.size(-1);
    ld = c;
    if (t.is_contiguous()) return;
    if (t.stride(-1) != 1 && c > 1) t = t.contiguous();
    t = t.reshape({-1, c});
    if (t.size(0) <= 1) return;
    if (t.stride(0) < c) t = t.contiguous();  // rows that overlap (an expanded tensor)
    ld = t.stride(0);
  }
};
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kHalf ? MHC_F16 : MHC_BF16; }

// y, and with keep_z the pre-activation in fp32, in rows padded to a multiple of 8.
Tensor linear_fwd(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& residual,
                  int act, bool keep_z, Tensor* z) {
  const c10::cuda::CUDAGuard on(x.device());
  const int64_t N = w.size(0), K = w.size(1), M = x.numel() / K;
  const Rows xr(x), wr(w), rr(residual);
  const Tensor b = bias.defined() ? bias.resolve_neg().contiguous() : bias;
  auto shape = x.sizes().vec();
  shape.back() = N;
  Tensor y = at::empty(shape, x.options());
  const int64_t ldz = (N + 7) / 8 * 8;
  if (keep_z) *z = at::empty({M, ldz}, x.options().dtype(at::kFloat));
  const size_t bytes = lib.fwd_bytes(ptr(xr.t), xr.ld, ptr(wr.t), wr.ld, M, N, K);
  const Tensor ws = workspace(bytes, x);
  check(lib.fwd(ptr(xr.t), xr.ld, ptr(wr.t), wr.ld, ptr(b), ptr(rr.t), rr.ld, dtype_of(x), act,
                keep_z ? z->data_ptr<float>() : nullptr, ldz, ptr(y), N, M, N, K, ptr(ws), bytes, stream_of(x)),
        "mhc_linear_fwd");
  return y;
}

struct Linear : torch::autograd::Function<Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w,
                        const std::optional<Tensor>& bias, const std::optional<Tensor>& residual,
                        int64_t act, bool wants) {
    Tensor z;
    Tensor y = linear_fwd(x, w, bias.value_or(Tensor()), residual.value_or(Tensor()), (int)act,
                          wants && act != 0, &z);
    ctx->save_for_backward({x, w, z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["operands"] = (int64_t)(2 + (bias ? 1 : 0));
    ctx->saved_data["residual"] = residual.has_value();
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &z = saved[2], &dy = grads[0];
    const int act = (int)ctx->saved_data["act"].toInt();
    const size_t operands = (size_t)ctx->saved_data["operands"].toInt();
    const bool has_bias = operands == 3;
    const bool want_dx = ctx->needs_input_grad(0), want_dw = ctx->needs_input_grad(1);
    const bool want_db = has_bias && ctx->needs_input_grad(2);
    Tensor dx, dw, db, dr;
    if (dy.defined()) require_no_tangent(dy);
    if (want_dx || want_dw || want_db) {
      const bool twice = at::GradMode::is_enabled();
      const at::AutoGradMode off(false);
      const c10::cuda::CUDAGuard on(x.device());
      const int64_t N = w.size(0), K = w.size(1), M = x.numel() / K;
      const Rows dr2(dy), xr(x), wr(w);
      if (want_dx) dx = at::empty(x.sizes(), x.options());
      if (want_dw) dw = at::empty({N, K}, x.options());
      if (want_db) db = at::empty({N}, x.options());
      const size_t bytes = lib.bwd_bytes(ptr(dr2.t), dr2.ld, ptr(xr.t), xr.ld, ptr(wr.t), wr.ld, act,
                                         want_dx, want_dw, want_db, M, N, K);
      const Tensor ws = workspace(bytes, x);
      check(lib.bwd(ptr(dr2.t), dr2.ld, z.defined() ? z.data_ptr<float>() : nullptr,
                    z.defined() ? z.size(1) : 0, ptr(xr.t), xr.ld,
                    ptr(wr.t), wr.ld, dtype_of(x), act, ptr(dx), K, ptr(dw), K, ptr(db), M, N, K,
                    ptr(ws), bytes, stream_of(x)),
            "mhc_linear_bwd");
      if (twice) {  // the gradients have no gradient: asking for one is an error
        const auto error = std::make_shared<torch::autograd::Error>(
            "linear_act can be differentiated once only",
            torch::autograd::collect_next_edges(x, w, dy));
        for (Tensor* t : {&dx, &dw, &db})
          if (t->defined()) torch::autograd::create_gradient_edge(*t, error);
      }
    }
    if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(operands)) dr = dy;
    return {dx, dw, db, dr, Tensor(), Tensor()};
  }
};

// linear(x, weight, bias or None, residual or None, act) -> Tensor
// Shapes and types have been checked.
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const Args in("linear", args, nargs, 5);
  const Tensor &x = in.tensor(0), &w = in.tensor(1);
  const Tensor b = in.maybe(2), r = in.maybe(3);
  const int64_t act = in.integer(4);
  require_cuda(x, {&w, &b, &r});
  Tensor y;
  {
    const pybind11::gil_scoped_release unlocked;
    const auto needs = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
    const auto given = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    const bool wants = needs(x) || needs(w) || needs(b);
    if (at::GradMode::is_enabled() && (wants || needs(r)))
      y = Linear::apply(x, w, given(b), given(r), act, wants);
    else  // a decoding step: nothing to record
      y = linear_fwd(x, w, b, r, (int)act, false, nullptr);
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// ----------------------------------------------------------------- losses --
// Logits [T, V] or [B, S, V] and their targets as the C ABI takes them: rows are
// read in place where the last axis is contiguous, else copied.
struct LogitRows {
  Tensor logits, targets;
  int64_t rows, per, batch_stride = 0, row_stride, V, ignore;
  int dtype;
  LogitRows(const Tensor& x, const Tensor& y, int64_t ignore_) : ignore(ignore_) {
    V = x.size(-1);
    logits = x.resolve_neg();
    if (logits.stride(-1) != 1 && V > 1) logits = logits.contiguous();
    targets = y.contiguous();
    rows = targets.numel();
    per = rows;
    row_stride = logits.stride(-2);
    if (logits.dim() == 3) {
      per = logits.size(1);
      batch_stride = logits.stride(0);
    }
    if (per < 1) per = 1;
    dtype = logits.scalar_type() == at::kFloat ? MHC_F32
            : logits.scalar_type() == at::kHalf ? MHC_F16
                                                : MHC_BF16;
  }
  Tensor floats(at::IntArrayRef shape) const {
    return at::empty(shape, logits.options().dtype(at::kFloat));
  }
  // as logits, contiguous
  Tensor gradient() const { return at::empty(logits.sizes(), logits.options()); }
};
Tensor f32(const Tensor& t) {
  return t.defined() ? t.to(at::kFloat).resolve_neg().contiguous() : t;
}
float* at_float(const Tensor& t, int64_t i = 0) {
  return t.defined() ? t.data_ptr<float>() + i : nullptr;
}

// token_logprobs(logits, targets, ignore) -> (logp, stats [4 rows])
PyObject* token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const Args in("token_logprobs", args, nargs, 3);
  const Tensor &x = in.tensor(0), &y = in.tensor(1);
  const int64_t ignore = in.integer(2);
  require_cuda(x, {&y});
  Tensor logp, stats;
  {
    const pybind11::gil_scoped_release unlocked;
    const at::AutoGradMode off(false);
    const c10::cuda::CUDAGuard on(x.device());
    const LogitRows r(x, y, ignore);
    logp = r.floats(y.sizes());
    stats = r.floats({4 * r.rows});
    check(lib.token_logprobs(ptr(r.logits), r.dtype, r.rows, r.per, r.batch_stride, r.row_stride, r.V,
                             r.targets.data_ptr<int64_t>(), r.ignore, at_float(logp), at_float(stats),
                             stream_of(x)),
          "mhc_token_logprobs");
  }
  return tuple_of({logp, stats});
  END_HANDLE_TH_ERRORS
}

// logits_grad(logits, targets, ignore, stats, coef or None, scale or None, ready or None)
//   -> coef * scale * (one-hot - softmax)
// coef None: it follows the stats, as a loss leaves them.  scale: a device scalar.
// ready: that gradient for a scale of 1, returned and overwritten unless the scale is 1.
PyObject* logits_grad(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const Args in("logits_grad", args, nargs, 7);
  const Tensor &x = in.tensor(0), &y = in.tensor(1), &stats = in.tensor(3);
  const Tensor coef = in.maybe(4), scale = in.maybe(5), ready = in.maybe(6);
  const int64_t ignore = in.integer(2);
  require_cuda(x, {&y, &stats, &coef, &scale, &ready});
  Tensor out;
  {
    const pybind11::gil_scoped_release unlocked;
    const at::AutoGradMode off(false);
    const c10::cuda::CUDAGuard on(x.device());
    const LogitRows r(x, y, ignore);
    const Tensor c = f32(coef), k = f32(scale);
    out = ready.defined() ? ready : r.gradient();
    check(lib.logits_grad(ptr(r.logits), r.dtype, r.rows, r.per, r.batch_stride, r.row_stride, r.V,
                          r.targets.data_ptr<int64_t>(), r.ignore, at_float(stats),
                          c.defined() ? at_float(c) : at_float(stats, 4 * r.rows), 1.0f, at_float(k),
                          ready.defined(), ptr(out), stream_of(x)),
          "mhc_logits_grad");
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// preference(logits, targets, ignore, ref, cu_seqlens or None, pairs, beta, smoothing,
//            inverse denominator, grad_scale, want_grad)
//   -> (loss, logp, margins, dlogits or None, stats and coef [5 rows])
PyObject* preference(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const Args in("preference", args, nargs, 11);
  const Tensor &x = in.tensor(0), &y = in.tensor(1), &ref = in.tensor(3);
  const Tensor cu = in.maybe(4);
  const int64_t ignore = in.integer(2), pairs = in.integer(5), want = in.integer(10);
  const float beta = in.number(6), smoothing = in.number(7), inv_d = in.number(8), scale = in.number(9);
  require_cuda(x, {&y, &ref, &cu});
  Tensor loss, logp, margins, dlogits, records;
  {
    const pybind11::gil_scoped_release unlocked;
    const at::AutoGradMode off(false);
    const c10::cuda::CUDAGuard on(x.device());
    const LogitRows r(x, y, ignore);
    const Tensor f = f32(ref), c = cu.defined() ? cu.contiguous() : cu;
    loss = r.floats({});
    logp = r.floats(y.sizes());
    margins = r.floats({pairs});
    records = r.floats({5 * r.rows});
    if (want) dlogits = r.gradient();
    check(lib.preference(ptr(r.logits), r.dtype, r.rows, r.per, r.batch_stride, r.row_stride, r.V,
                         r.targets.data_ptr<int64_t>(), r.ignore, ptr(c),
                         c.defined() && c.scalar_type() == at::kLong, c.defined() ? 0 : r.logits.size(1),
                         pairs, at_float(f), beta, smoothing, inv_d, scale, at_float(logp),
                         at_float(records), at_float(records, 4 * r.rows), at_float(margins),
                         at_float(loss), ptr(dlogits), stream_of(x)),
          "mhc_preference_loss");
  }
  return tuple_of({loss, logp, margins, dlogits, records});
  END_HANDLE_TH_ERRORS
}

// policy(logits, targets, ignore, old, advantages, ref or None, clip_low, clip_high, kl_coef,
//        inverse denominator or 0, grad_scale, want_grad)
//   -> (loss, logp, kl, dlogits or None, stats and coef [5 rows])
PyObject* policy(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const Args in("policy", args, nargs, 12);
  const Tensor &x = in.tensor(0), &y = in.tensor(1), &old = in.tensor(3), &adv = in.tensor(4);
  const Tensor ref = in.maybe(5);
  const int64_t ignore = in.integer(2), want = in.integer(11);
  const float lo = in.number(6), hi = in.number(7), kl_coef = in.number(8), inv_d = in.number(9),
              scale = in.number(10);
  require_cuda(x, {&y, &old, &adv, &ref});
  Tensor loss, logp, kl, dlogits, records;
  {
    const pybind11::gil_scoped_release unlocked;
    const at::AutoGradMode off(false);
    const c10::cuda::CUDAGuard on(x.device());
    const LogitRows r(x, y, ignore);
    const Tensor o = f32(old), a = f32(adv), f = f32(ref);
    loss = r.floats({});
    kl = r.floats({});
    logp = r.floats(y.sizes());
    records = r.floats({5 * r.rows});
    if (want) dlogits = r.gradient();
    const size_t bytes = lib.policy_bytes();
    const Tensor ws = workspace(bytes, x);
    check(lib.policy(ptr(r.logits), r.dtype, r.rows, r.per, r.batch_stride, r.row_stride, r.V,
                     r.targets.data_ptr<int64_t>(), r.ignore, at_float(o), at_float(a), at_float(f), lo,
                     hi, kl_coef, inv_d, scale, at_float(logp), at_float(records),
                     at_float(records, 4 * r.rows), at_float(loss), at_float(kl), ptr(dlogits), ptr(ws),
                     bytes, stream_of(x)),
          "mhc_policy_loss");
  }
  return tuple_of({loss, logp, kl, dlogits, records});
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the entry points of Library, in their order, MHCError)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  constexpr int n = sizeof(Library) / sizeof(void*);
  void* p[n];
  if (nargs != n + 1 || !PyExceptionClass_Check(args[n])) {
    PyErr_Format(PyExc_TypeError, "bind: %d addresses and an exception are expected", n);
    return nullptr;
  }
  for (int i = 0; i < n; ++i) p[i] = PyLong_AsVoidPtr(args[i]);
  if (PyErr_Occurred()) return nullptr;
  static_assert(sizeof(Library) == sizeof(p), "one address a member");
  std::memcpy(&lib, p, sizeof(p));
  Py_XSETREF(mhc_error, Py_NewRef(args[n]));
  Py_RETURN_NONE;
}

// ----------------------------------------------------------------- gather --

// The same codes as the C ABI's.
bool type_of(int code, at::ScalarType* t) {
  if (code == 0) *t = at::kFloat;
  else if (code == 1) *t = at::kHalf;
  else if (code == 2) *t = at::kBFloat16;
  else return false;
  return true;
}

bool as_laid_out(const Tensor& t, at::ScalarType type, c10::DeviceIndex device, int64_t numel) {
  return t.defined() && t.layout() == at::kStrided && t.is_cuda() && t.device().index() == device &&
         t.scalar_type() == type && t.numel() == numel && t.is_contiguous() && !t.is_neg();
}

// gather(params, numel, dtype, device, p_out, g_out) -> bool
// params: a list; numel (int64), p_out, g_out (uint64): addresses of arrays as long.
// True: every parameter and its gradient is a plain contiguous CUDA tensor of that
// type, device and size, and its address has been written.  False: one is not.
PyObject* gather(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 6 || !PyList_CheckExact(args[0])) {
    PyErr_SetString(PyExc_TypeError, "gather(params: list, numel, dtype, device, p_out, g_out)");
    return nullptr;
  }
  const auto* numel = static_cast<const int64_t*>(PyLong_AsVoidPtr(args[1]));
  const long code = PyLong_AsLong(args[2]), device = PyLong_AsLong(args[3]);
  auto* p_out = static_cast<uint64_t*>(PyLong_AsVoidPtr(args[4]));
  auto* g_out = static_cast<uint64_t*>(PyLong_AsVoidPtr(args[5]));
  if (PyErr_Occurred()) return nullptr;
  at::ScalarType type;
  if (!numel || !p_out || !g_out || device < 0 || device > 127 || !type_of((int)code, &type)) {
    PyErr_SetString(PyExc_ValueError, "gather: a missing array, or a bad dtype or device");
    return nullptr;
  }
  try {
    const Py_ssize_t n = PyList_GET_SIZE(args[0]);
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = PyList_GET_ITEM(args[0], i);
      if (!THPVariable_CheckExact(o)) Py_RETURN_FALSE;  // a subclass answers for itself
      const Tensor& p = THPVariable_Unpack(o);
      if (!as_laid_out(p, type, (c10::DeviceIndex)device, numel[i])) Py_RETURN_FALSE;
      const Tensor& g = p.unsafeGetTensorImpl()->grad();
      if (!as_laid_out(g, type, (c10::DeviceIndex)device, numel[i])) Py_RETURN_FALSE;
      p_out[i] = (uint64_t) reinterpret_cast<uintptr_t>(p.mutable_data_ptr());
      g_out[i] = (uint64_t) reinterpret_cast<uintptr_t>(g.const_data_ptr());
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "gather: an unknown C++ exception");
    return nullptr;
  }
  Py_RETURN_TRUE;
}

// changed(tensors): a list of tensors whose values a kernel has written through their
// addresses.  Their versions go up, as a torch operation in place would raise them: a
// graph that saved one of them can tell.
PyObject* changed(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const Args in("changed", args, nargs, 1);
  TORCH_CHECK_TYPE(PyList_CheckExact(args[0]), "changed: a list is expected");
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(args[0]); ++i) {
    PyObject* o = PyList_GET_ITEM(args[0], i);
    TORCH_CHECK_TYPE(THPVariable_Check(o), "changed: a list of tensors is expected");
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();  // those have no version
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}
PyMethodDef methods[] = {
    {"bind", fast(bind), METH_FASTCALL, "bind(the entry points' addresses, MHCError)"},
    {"token_logprobs", fast(token_logprobs), METH_FASTCALL, "-> (logp, stats)"},
    {"logits_grad", fast(logits_grad), METH_FASTCALL, "-> dlogits"},
    {"preference", fast(preference), METH_FASTCALL, "-> (loss, logp, margins, dlogits, records)"},
    {"policy", fast(policy), METH_FASTCALL, "-> (loss, logp, kl, dlogits, records)"},
    {"linear", fast(linear), METH_FASTCALL, "linear(x, weight, bias, residual, act) -> Tensor"},
    {"gather", fast(gather), METH_FASTCALL,
     "gather(params, numel, dtype, device, p_out, g_out) -> bool"},
    {"changed", fast(changed), METH_FASTCALL, "changed(tensors): raises their versions"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mhc_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__mhc_host() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "build_id", MHC_HOST_ID) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
