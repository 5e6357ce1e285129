// What an optimizer step asks of hundreds of tensors, in one call from Python:
// 512 parameters' and gradients' sizes, types, devices, layouts and addresses
// take some 250 us one attribute at a time from Python and 10 us here.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/python_variable.h>

namespace {

// The same codes as the C ABI's.
bool type_of(int code, at::ScalarType* t) {
  if (code == 0) *t = at::kFloat;
  else if (code == 1) *t = at::kHalf;
  else if (code == 2) *t = at::kBFloat16;
  else return false;
  return true;
}

bool as_laid_out(const at::Tensor& t, at::ScalarType type, c10::DeviceIndex device, int64_t numel) {
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
      const at::Tensor& p = THPVariable_Unpack(o);
      if (!as_laid_out(p, type, (c10::DeviceIndex)device, numel[i])) Py_RETURN_FALSE;
      const at::Tensor& g = p.unsafeGetTensorImpl()->grad();
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

PyMethodDef methods[] = {
    {"gather", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gather)), METH_FASTCALL,
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
