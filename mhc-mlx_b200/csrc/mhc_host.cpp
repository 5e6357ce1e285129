// The parts of two operators that run on the host for every call and took longer
// from Python than their kernels do.
//
//   gather   what an optimizer step asks of hundreds of tensors: 512 parameters'
//            and gradients' sizes, types, devices, layouts and addresses take
//            some 250 us one attribute at a time, 10 us here.
//   linear   the linear layer over the C ABI, and its place in autograd: the
//            engine calls a backward that is written in Python with the
//            interpreter's lock, on a thread of its own.
#include <Python.h>

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
  decltype(&mhc_last_error) last_error;
} lib = {};

void check(int status, const char* fn) {
  if (status == MHC_OK) return;
  TORCH_CHECK_VALUE(status != MHC_ERR_INVALID, fn, ": ", lib.last_error());
  TORCH_CHECK(false, fn, " failed (status ", status, "): ", lib.last_error());
}
void* stream_of(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor workspace(size_t bytes, const Tensor& like) {
  if (bytes == 0) return {};
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
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

// y, and with keep_z the pre-activation in rows padded to a multiple of 8.
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
  if (keep_z) *z = at::empty({M, ldz}, x.options());
  const size_t bytes = lib.fwd_bytes(ptr(xr.t), xr.ld, ptr(wr.t), wr.ld, M, N, K);
  const Tensor ws = workspace(bytes, x);
  check(lib.fwd(ptr(xr.t), xr.ld, ptr(wr.t), wr.ld, ptr(b), ptr(rr.t), rr.ld, dtype_of(x), act,
                keep_z ? ptr(*z) : nullptr, ldz, ptr(y), N, M, N, K, ptr(ws), bytes, stream_of(x)),
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
      check(lib.bwd(ptr(dr2.t), dr2.ld, ptr(z), z.defined() ? z.size(1) : 0, ptr(xr.t), xr.ld,
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
  TORCH_CHECK_TYPE(nargs == 5 && THPVariable_Check(args[0]) && THPVariable_Check(args[1]) &&
                       (args[2] == Py_None || THPVariable_Check(args[2])) &&
                       (args[3] == Py_None || THPVariable_Check(args[3])) && PyLong_Check(args[4]),
                   "linear(x, weight, bias, residual, act): tensors and an int are expected");
  const Tensor &x = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]);
  std::optional<Tensor> bias, residual;
  if (args[2] != Py_None) bias = THPVariable_Unpack(args[2]);
  if (args[3] != Py_None) residual = THPVariable_Unpack(args[3]);
  const long act = PyLong_AsLong(args[4]);
  if (PyErr_Occurred()) return nullptr;
  TORCH_CHECK(lib.fwd != nullptr, "the library is not loaded");
  for (const Tensor* t : {&x, &w, bias ? &*bias : &x, residual ? &*residual : &x}) {
    TORCH_CHECK(t->is_cuda(), "mhc_b200 runs only on CUDA tensors (sm_100a kernels); got a tensor on ",
                t->device(), ".  There is no CPU fallback.");
    TORCH_CHECK_VALUE(t->device() == x.device(), "tensors on different devices: ", x.device(), " and ",
                      t->device());
  }
  Tensor y;
  {
    const pybind11::gil_scoped_release unlocked;
    const auto needs = [](const std::optional<Tensor>& t) { return t && t->requires_grad(); };
    const bool wants = x.requires_grad() || w.requires_grad() || needs(bias);
    if (at::GradMode::is_enabled() && (wants || needs(residual)))
      y = Linear::apply(x, w, bias, residual, (int64_t)act, wants);
    else  // a decoding step: nothing to record
      y = linear_fwd(x, w, bias.value_or(Tensor()), residual.value_or(Tensor()), (int)act, false, nullptr);
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the entry points above, in their order)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  void* p[5];
  if (nargs != 5) {
    PyErr_SetString(PyExc_TypeError, "bind: five addresses are expected");
    return nullptr;
  }
  for (int i = 0; i < 5; ++i) p[i] = PyLong_AsVoidPtr(args[i]);
  if (PyErr_Occurred()) return nullptr;
  lib = {reinterpret_cast<decltype(lib.fwd_bytes)>(p[0]), reinterpret_cast<decltype(lib.fwd)>(p[1]),
         reinterpret_cast<decltype(lib.bwd_bytes)>(p[2]), reinterpret_cast<decltype(lib.bwd)>(p[3]),
         reinterpret_cast<decltype(lib.last_error)>(p[4])};
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

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}
PyMethodDef methods[] = {
    {"bind", fast(bind), METH_FASTCALL, "bind(five entry points' addresses)"},
    {"linear", fast(linear), METH_FASTCALL, "linear(x, weight, bias, residual, act) -> Tensor"},
    {"gather", fast(gather), METH_FASTCALL,
     "gather(params, numel, dtype, device, p_out, g_out) -> bool"},
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
