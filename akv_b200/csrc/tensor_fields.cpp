// fields(ndim, tensor, ...) -> one flat tuple with, per tensor, its address,
// device index (-1: the CPU), type code, sizes and strides.
//
// The Python wrappers check shapes, types, strides and devices of up to a dozen
// tensors per call; asking a tensor for each of them costs about 1.2 us a tensor,
// this 0.17 (a qk_norm_rope call of one token: 15.2 us of host time, now 9.9).
// A CPython module because only it sees the tensors; the kernels' library keeps
// its plain C ABI.

#include <torch/csrc/autograd/python_variable.h>

namespace {

PyObject* fields(PyObject*, PyObject* const* args, Py_ssize_t n) {
  const long ndim = n > 0 ? PyLong_AsLong(args[0]) : -1;
  if (ndim < 0 || ndim > 8) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "fields(ndim, tensor, ...)");
    return nullptr;
  }
  PyObject* out = PyTuple_New((n - 1) * (3 + 2 * ndim));
  if (out == nullptr) return nullptr;
  Py_ssize_t at = 0;
  bool ok = true;
  auto put = [&](long long x) {
    PyObject* v = PyLong_FromLongLong(x);
    ok = ok && v != nullptr;
    PyTuple_SET_ITEM(out, at++, v);
  };
  try {
    for (Py_ssize_t i = 1; i < n && ok; ++i) {
      if (!THPVariable_Check(args[i])) {
        PyErr_Format(PyExc_ValueError, "argument %zd is no tensor", i);
        ok = false;
        break;
      }
      const at::Tensor& t = THPVariable_Unpack(args[i]);
      if (t.dim() != ndim) {
        PyErr_Format(PyExc_ValueError, "a tensor of %ld dimensions where %ld are needed",
                     (long)t.dim(), ndim);
        ok = false;
        break;
      }
      put((long long)reinterpret_cast<intptr_t>(t.data_ptr()));
      put(t.get_device());
      put((long long)t.scalar_type());
      for (long k = 0; k < ndim; ++k) put(t.size(k));
      for (long k = 0; k < ndim; ++k) put(t.stride(k));
    }
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, e.what());
    ok = false;
  }
  if (!ok) {
    Py_DECREF(out);
    return nullptr;
  }
  return out;
}

PyMethodDef methods[] = {
    {"fields", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(fields)), METH_FASTCALL,
     "fields(ndim, tensor, ...): address, device, type, sizes and strides of each"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_fields", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_fields(void) {
  PyObject* m = PyModule_Create(&module);
  if (m == nullptr) return nullptr;
  // The tensor's layout is that of this torch: _native checks it.
  PyModule_AddStringConstant(m, "BUILT_FOR", AKV_TORCH_VERSION);
  PyModule_AddIntConstant(m, "INT32", (long)at::kInt);
  PyModule_AddIntConstant(m, "INT64", (long)at::kLong);
  PyModule_AddIntConstant(m, "F16", (long)at::kHalf);
  PyModule_AddIntConstant(m, "BF16", (long)at::kBFloat16);
  PyModule_AddIntConstant(m, "F32", (long)at::kFloat);
  return m;
}
