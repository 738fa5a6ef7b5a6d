// Host-side walk over a list of tensors for the multi-tensor operators: what a Python loop spends
// half a microsecond a tensor on (gradient, address, size, type, device, order of dimensions) in one
// call.  A CPython extension module, retinahead._host.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>
#include <string>
#include "retinahead.h"

namespace {

// (device index, bytes of rh_tensor_ref [count]), or a text that says what is wrong with the list.
// An empty list gives (-1, b"").
PyObject* table_of(PyObject* list, const bool grads) {
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(list);
  PyObject** items = PySequence_Fast_ITEMS(list);
  std::string refs;
  refs.reserve((size_t)n * sizeof(rh_tensor_ref));
  int device = -1;
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (!THPVariable_Check(items[i])) return PyUnicode_FromString("a list of tensors is needed");
    const at::Tensor& item = THPVariable_Unpack(items[i]);
    const at::Tensor t = grads ? item.grad() : item;
    if (!t.defined()) continue;
    if (t.layout() != at::kStrided) return PyUnicode_FromString("gradients must be dense tensors, not sparse ones");
    if (!t.is_cuda())
      return PyUnicode_FromString("retinahead operators need tensors on a HIP device (there is no CPU fallback)");
    if (device < 0) device = t.get_device();
    if (t.get_device() != device) return PyUnicode_FromString("tensors on different devices");
    rh_tensor_ref r = {};
    switch (t.scalar_type()) {
      case at::kFloat: r.dtype = RH_F32; break;
      case at::kBFloat16: r.dtype = RH_BF16; break;
      case at::kHalf: r.dtype = RH_F16; break;
      default: return PyUnicode_FromString("float32, bfloat16 or float16 tensors needed");
    }
    if (!t.is_non_overlapping_and_dense())
      return PyUnicode_FromString("gradients must fill their memory: a strided or expanded view does not");
    r.count = t.numel();
    r.data = r.count ? const_cast<void*>(t.const_data_ptr()) : nullptr;
    refs.append(reinterpret_cast<const char*>(&r), sizeof(r));
  }
  return Py_BuildValue("(iy#)", device, refs.data(), (Py_ssize_t)refs.size());
}

PyObject* tensor_table(PyObject*, PyObject* args) {
  PyObject* list = nullptr;
  int grads = 0;
  if (!PyArg_ParseTuple(args, "Op", &list, &grads)) return nullptr;
  PyObject* fast = PySequence_Fast(list, "a list of tensors is needed");
  if (!fast) return nullptr;
  PyObject* out = nullptr;
  try {
    out = table_of(fast, grads != 0);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  Py_DECREF(fast);
  return out;
}

PyMethodDef methods[] = {
    {"tensor_table", tensor_table, METH_VARARGS,
     "tensor_table(tensors, grads): (device index, table) of the tensors, or of their gradients; a str says what is wrong"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Host-side walk over lists of tensors.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__host(void) { return PyModule_Create(&module); }
