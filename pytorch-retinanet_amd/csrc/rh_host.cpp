// What Python is slow at on the way to the operators' entry points.  A CPython extension module,
// retinahead._host.
//   - The walk over a list of tensors for the multi-tensor operators (gradient, address, size, type, device,
//     order of dimensions): half a microsecond a tensor in a Python loop.
//   - The classifier loss's checks, outputs and autograd node.  16 x 256 rows against 80 classes, forward and
//     backward: 116 us on the host in Python, 58 here; a scaled sum of four values takes 54.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <array>
#include <atomic>
#include <map>
#include <memory>
#include <mutex>
#include <string>
#include "retinahead.h"

namespace {

int type_code(const at::ScalarType t) {      // -1: not one of the operators' types
  switch (t) {
    case at::kFloat: return RH_F32;
    case at::kBFloat16: return RH_BF16;
    case at::kHalf: return RH_F16;
    default: return -1;
  }
}
const char* const kTypes = "float32, bfloat16 or float16 tensors needed";
// a tangent would be dropped, which counts as zero
const char* const kNoTangents = "retinahead operators do not support forward-mode differentiation";
const char* const kNoFallback = "retinahead operators need tensors on a HIP device (there is no CPU fallback)";

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
    if (t._fw_grad(0).defined()) return PyUnicode_FromString(kNoTangents);
    if (t.layout() != at::kStrided) return PyUnicode_FromString("gradients must be dense tensors, not sparse ones");
    if (!t.is_cuda())
      return PyUnicode_FromString(kNoFallback);
    if (device < 0) device = t.get_device();
    if (t.get_device() != device) return PyUnicode_FromString("tensors on different devices");
    rh_tensor_ref r = {};
    r.dtype = type_code(t.scalar_type());
    if (r.dtype < 0) return PyUnicode_FromString(kTypes);
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

// ---------------------------------------------------------------------------------------------
// Classifier loss
// ---------------------------------------------------------------------------------------------
struct Entry {      // what bind() was given
  size_t (*bytes)(int64_t, int32_t, int64_t, int32_t, int32_t) = nullptr;
  int (*run)(const rh_linear_ce_args*, void*) = nullptr;
  int (*scale)(void*, int64_t, int32_t, const float*, float, void*) = nullptr;
  size_t (*last_error)(char*, size_t) = nullptr;
  PyObject* workspace = nullptr;      // (device, bytes, tag, stream) -> tensor
  PyObject* error = nullptr;          // RetinaHeadError
} entry;

constexpr int kDevices = 64;
std::atomic<const void*> unit[kDevices];      // address of each device's tensor that is known to hold 1.0

std::string last_error() {
  char text[512] = "";
  entry.last_error(text, sizeof(text));
  return text;
}

struct Refusal {
  std::string text;
};
void refuse_unless(const bool ok, const char* text) {
  if (!ok) throw Refusal{text};
}

void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

struct WithInterpreter {
  const PyGILState_STATE state = PyGILState_Ensure();
  ~WithInterpreter() { PyGILState_Release(state); }
};

// In a node's backward: RetinaHeadError for the caller of backward().
[[noreturn]] void raise_in_backward(const std::string& text) {
  python_error e;
  {
    const WithInterpreter held;
    PyErr_SetString(entry.error, text.c_str());
    e.persist();
  }
  throw e;
}

struct CeOut {
  at::Tensor small, row_loss;
  std::array<at::Tensor, 3> grads;
};

struct Settings {
  long long ignore_index;
  int reduction;
  double expected;
};

// Under the interpreter's lock.  made: gradients of an earlier call with these arguments, to be made again where the
// upstream gradient is not the expected one.
CeOut classifier_loss(const at::Tensor& features, const at::Tensor& weight, const at::Tensor& labels,
                      const at::Tensor& bias, const at::Tensor& divisor, const Settings& q,
                      const std::array<bool, 3>& want, const std::array<at::Tensor, 3>& made = {},
                      const at::Tensor& upstream = {}) {
  for (const at::Tensor* t : {&features, &weight, &bias, &divisor})
    refuse_unless(!t->defined() || !t->_fw_grad(0).defined(), kNoTangents);
  at::AutoDispatchBelowAutograd below;
  const int code = type_code(features.scalar_type());
  refuse_unless(code >= 0, kTypes);
  refuse_unless(weight.scalar_type() == features.scalar_type() &&
                    (!bias.defined() || bias.scalar_type() == features.scalar_type()),
                "features, weight and bias must have one element type");
  refuse_unless(weight.dim() == 2 && features.dim() >= 1 && features.size(-1) == weight.size(1),
                "expected features [..., D] and weight [V, D]");
  refuse_unless(labels.sizes() == features.sizes().slice(0, features.dim() - 1),
                "labels must have the features' shape without the last dimension");
  refuse_unless(labels.scalar_type() == at::kLong || labels.scalar_type() == at::kInt, "labels must be int64 or int32");
  const int64_t v = weight.size(0), d = weight.size(1), n = labels.numel();
  refuse_unless(!bias.defined() || (bias.dim() == 1 && bias.size(0) == v), "bias must be [V]");
  refuse_unless(v >= 1 && d >= 1, "linear_cross_entropy needs at least one class and one feature");
  refuse_unless(!divisor.defined() || (divisor.scalar_type() == at::kFloat && divisor.numel() == 1),
                "divisor must be one float32");
  const c10::Device device = features.device();
  for (const at::Tensor* t : {&features, &weight, &labels, &bias, &divisor}) {
    if (!t->defined()) continue;
    refuse_unless(t->is_cuda() && t->layout() == at::kStrided, kNoFallback);
    if (t->device() != device)
      throw Refusal{"tensors on different devices: " + device.str() + " and " + t->device().str()};
  }
  c10::DeviceGuard on(device);
  const at::TensorOptions as_features = at::TensorOptions().dtype(features.scalar_type()).device(device);
  const at::TensorOptions floats = at::TensorOptions().dtype(at::kFloat).device(device);
  CeOut out;
  out.grads = made;
  out.small = at::empty({4}, floats);
  out.row_loss = at::empty(labels.sizes(), floats);
  if (want[0]) out.grads[0] = at::empty(features.sizes(), as_features);
  if (want[1]) out.grads[1] = at::empty({v, d}, as_features);
  if (want[2] && bias.defined()) out.grads[2] = at::empty({v}, as_features);
  if (n == 0) {
    out.small.zero_();
    for (at::Tensor& t : out.grads)
      if (t.defined()) t.zero_();
    return out;
  }
  at::Tensor x = features.dim() == 2 ? features : features.reshape({n, d});
  if (x.stride(1) != 1 || x.stride(0) < d) x = x.contiguous();
  at::Tensor w = weight;
  if (w.stride(1) != 1 || w.stride(0) < d) w = w.contiguous();
  const at::Tensor y = labels.contiguous(), b = bias.defined() ? bias.contiguous() : bias;
  const int64_t size = w.element_size();
  rh_linear_ce_args a = {};
  a.x = x.const_data_ptr();
  a.w = w.const_data_ptr();
  a.bias = b.defined() ? b.const_data_ptr() : nullptr;
  a.labels = y.const_data_ptr();
  a.n = n;
  a.v = v;
  a.ldx = n > 1 ? x.stride(0) : d;
  a.ldw = v > 1 ? w.stride(0) : std::max(d, w.stride(0));
  refuse_unless(d <= INT32_MAX, "too many features");
  a.d = (int32_t)d;
  a.dtype = code;
  a.labels_int64 = y.scalar_type() == at::kLong;
  a.reduction = q.reduction;
  a.ignore_index = q.ignore_index;
  a.divisor = divisor.defined() ? divisor.const_data_ptr<float>() : nullptr;
  a.upstream = upstream.defined() ? upstream.const_data_ptr<float>() : nullptr;
  a.grad = (float)q.expected;
  a.flags = d * size % 16 || w.stride(0) * size % 16 || (uintptr_t)a.w % 16 || w.stride(0) >= 1 << 20
                ? RH_CE_COPY_WEIGHT : 0;
  a.row_loss = out.row_loss.data_ptr<float>();
  a.small = out.small.data_ptr<float>();
  a.dx = out.grads[0].defined() ? out.grads[0].data_ptr() : nullptr;
  a.dw = out.grads[1].defined() ? out.grads[1].data_ptr() : nullptr;
  a.db = out.grads[2].defined() ? out.grads[2].data_ptr() : nullptr;
  const int ask = a.flags | (a.dx ? RH_CE_GRAD_X : 0) | (a.dw ? RH_CE_GRAD_W : 0) | (a.db ? RH_CE_GRAD_B : 0);
  static std::map<std::array<int64_t, 5>, size_t> known;      // under the interpreter's lock
  if (known.size() >= 4096) known.clear();
  size_t& slot = known[{n, d, v, code, ask}];
  if (slot == 0) slot = entry.bytes(n, a.d, v, code, ask);
  const size_t need = slot;
  if (need == 0) throw Refusal{"linear_cross_entropy: " + last_error()};
  void* const stream = stream_of(features);
  PyObject* const py_device = THPDevice_New(device);
  if (!py_device) throw python_error();
  PyObject* const ws = PyObject_CallFunction(entry.workspace, "NnsK", py_device, (Py_ssize_t)need, "linear_ce",
                                             (unsigned long long)(uintptr_t)stream);
  if (!ws) throw python_error();
  const at::Tensor room = THPVariable_Unpack(ws);
  Py_DECREF(ws);
  a.workspace = room.data_ptr();
  a.workspace_bytes = room.numel();
  // under the interpreter's lock: two threads on one stream share the workspace, so a call's launches must not
  // fall between another's
  const int code_of_call = entry.run(&a, stream);
  if (code_of_call != RH_OK)
    throw Refusal{"rh_linear_ce failed (" + std::to_string(code_of_call) + "): " + last_error()};
  return out;
}

// The forward call makes the gradients, backward hands them out, times the upstream one where that is not
// the one they were made for.  float16 has no room for that: gradients made for 1 may be too small for it where those
// of a scaled loss are not (a mean over many rows), or too large, so there they are made anew from the inputs.
struct LinearCrossEntropyBackward : public torch::autograd::Node {
  std::array<at::Tensor, 3> grads;
  struct Inputs {      // features, weight, labels, bias, divisor; those made under inference mode as they are
    std::array<torch::autograd::SavedVariable, 5> saved;
    std::array<at::Tensor, 5> frozen;
  };
  std::unique_ptr<Inputs> inputs;      // float16
  Settings settings = {};
  bool spent = false;
  std::mutex once;

  std::string name() const override { return "LinearCrossEntropyBackward"; }

  torch::autograd::variable_list apply(torch::autograd::variable_list&& upstream) override {
    torch::autograd::variable_list out(3);
    std::array<at::Tensor, 5> of;
    bool anew = false;
    const at::Tensor& g = upstream[0];
    const bool as_made = settings.expected == 1.0 && g.defined() && g.numel() == 1 && g.is_cuda() &&
                         g.get_device() < kDevices && g.const_data_ptr() == unit[g.get_device()].load();
    {
      std::lock_guard<std::mutex> lock(once);
      if (spent)
        raise_in_backward("the fused loss keeps one set of gradients: backward() can run once per forward()");
      anew = inputs != nullptr && g.defined() && !as_made;
      if (anew)
        for (int i = 0; i < 5; ++i)      // unpack() refuses what was changed in place
          of[i] = inputs->frozen[i].defined() ? inputs->frozen[i] : inputs->saved[i].unpack();
      spent = true;
      for (int i = 0; i < 3; ++i) out[i] = std::move(grads[i]);
    }
    if (!g.defined()) return torch::autograd::variable_list(3);
    if (!as_made) {
      at::AutoDispatchBelowAutograd below;
      const at::Tensor scale = g.reshape({-1}).slice(0, 0, 1).to(at::kFloat).contiguous();
      if (anew)
        make_anew(of, scale, out);
      else
        for (const at::Tensor& d : out) {
          if (!d.defined()) continue;
          c10::DeviceGuard on(d.device());
          if (entry.scale(d.data_ptr(), d.numel(), type_code(d.scalar_type()), scale.const_data_ptr<float>(),
                          (float)settings.expected, stream_of(d)) != RH_OK)
            raise_in_backward("rh_scale_gradient failed: " + last_error());
        }
    }
    if (!at::GradMode::is_enabled()) return out;
    // create_graph: the gradients are there, their own gradients are not
    for (at::Tensor& d : out)
      if (d.defined()) d = d.detach().requires_grad_(true);
    return torch::autograd::DelayedError("the classifier loss's gradients cannot be differentiated", 3).apply(std::move(out));
  }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(once);
    for (at::Tensor& d : grads) d.reset();
    inputs.reset();
    spent = true;
  }

 private:
  void make_anew(const std::array<at::Tensor, 5>& of, const at::Tensor& scale, const torch::autograd::variable_list& out) {
    const WithInterpreter held;      // classifier_loss wants it
    try {
      classifier_loss(of[0], of[1], of[2], of[3], of[4], settings, {}, {out[0], out[1], out[2]}, scale);
    } catch (const Refusal& e) {
      raise_in_backward(e.text);
    } catch (python_error& e) {
      e.persist();
      throw;
    }
  }
};

bool tensor_or_none(PyObject* o, at::Tensor& t) {
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  t = THPVariable_Unpack(o);
  return true;
}

// tensors as a tuple; an undefined one is None
PyObject* as_tuple(std::initializer_list<at::Tensor> tensors) {
  PyObject* out = PyTuple_New((Py_ssize_t)tensors.size());
  if (!out) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : tensors) {
    PyObject* o = t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None);
    if (!o) {
      Py_DECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

PyObject* linear_ce(PyObject*, PyObject* args) {
  PyObject *o_features, *o_weight, *o_labels, *o_bias, *o_divisor;
  Settings q;
  int gx, gw, gb;
  PyObject* node;
  if (!PyArg_ParseTuple(args, "OOOOOLidpppO", &o_features, &o_weight, &o_labels, &o_bias, &o_divisor, &q.ignore_index,
                        &q.reduction, &q.expected, &gx, &gw, &gb, &node))
    return nullptr;
  try {
    at::Tensor features, weight, labels, bias, divisor;
    if (!tensor_or_none(o_features, features) || !tensor_or_none(o_weight, weight) || !tensor_or_none(o_labels, labels) ||
        !tensor_or_none(o_bias, bias) || !tensor_or_none(o_divisor, divisor) || !features.defined() ||
        !weight.defined() || !labels.defined()) {
      PyErr_SetString(PyExc_TypeError, "features, weight and labels must be tensors, bias and divisor tensors or None");
      return nullptr;
    }
    if (node != Py_None && !PyType_Check(node)) {
      PyErr_SetString(PyExc_TypeError, "node must be a class or None");
      return nullptr;
    }
    std::array<bool, 3> want = {gx != 0, gw != 0, gb != 0};
    if (node != Py_None) {
      const bool on = at::GradMode::is_enabled();
      want = {on && features.requires_grad(), on && weight.requires_grad(),
              on && bias.defined() && bias.requires_grad()};
    }
    CeOut out = classifier_loss(features, weight, labels, bias, divisor, q, want);
    if (node == Py_None) return as_tuple({out.small, out.row_loss, out.grads[0], out.grads[1], out.grads[2]});
    // on the small buffer's storage without being a view of it: views of a node's output refuse in-place operations
    at::Tensor loss;
    {
      at::AutoDispatchBelowAutograd below;
      loss = at::empty({0}, out.small.options());
      loss.set_(out.small.storage(), out.small.storage_offset(), {1}, {1});
    }
    if (want[0] || want[1] || want[2]) {
      auto made = std::shared_ptr<LinearCrossEntropyBackward>(new LinearCrossEntropyBackward(), torch::autograd::deleteNode);
      made->set_next_edges(torch::autograd::collect_next_edges(features, weight, bias));
      made->grads = std::move(out.grads);
      made->settings = q;
      if (features.scalar_type() == at::kHalf) {
        made->inputs = std::make_unique<LinearCrossEntropyBackward::Inputs>();
        const at::Tensor* const of[5] = {&features, &weight, &labels, &bias, &divisor};
        for (int i = 0; i < 5; ++i)
          if (of[i]->defined() && of[i]->is_inference()) made->inputs->frozen[i] = *of[i];
          else made->inputs->saved[i] = torch::autograd::SavedVariable(*of[i], false);
      }
      torch::autograd::set_history(loss, made);
    }
    PyObject* const as_class = THPVariable_Wrap(loss, reinterpret_cast<PyTypeObject*>(node));
    if (!as_class) return nullptr;
    PyObject* const rest = as_tuple({out.small, out.row_loss});
    if (!rest) {
      Py_DECREF(as_class);
      return nullptr;
    }
    return Py_BuildValue("(NN)", as_class, rest);
  } catch (const Refusal& e) {
    PyErr_SetString(entry.error ? entry.error : PyExc_RuntimeError, e.text.c_str());
  } catch (python_error& e) {
    e.restore();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long bytes, run, scale, error_text;
  PyObject *workspace, *error;
  if (!PyArg_ParseTuple(args, "KKKKOO", &bytes, &run, &scale, &error_text, &workspace, &error)) return nullptr;
  entry.bytes = (decltype(entry.bytes))(uintptr_t)bytes;
  entry.run = (decltype(entry.run))(uintptr_t)run;
  entry.scale = (decltype(entry.scale))(uintptr_t)scale;
  entry.last_error = (decltype(entry.last_error))(uintptr_t)error_text;
  entry.workspace = Py_NewRef(workspace);
  entry.error = Py_NewRef(error);
  Py_RETURN_NONE;
}

PyObject* know_unit(PyObject*, PyObject* args) {
  int device;
  unsigned long long at;
  if (!PyArg_ParseTuple(args, "iK", &device, &at)) return nullptr;
  if (device >= 0 && device < kDevices) unit[device] = (const void*)(uintptr_t)at;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"tensor_table", tensor_table, METH_VARARGS,
     "tensor_table(tensors, grads): (device index, table) of the tensors, or of their gradients; a str says what is wrong"},
    {"linear_ce", linear_ce, METH_VARARGS,
     "linear_ce(features, weight, labels, bias, divisor, ignore_index, reduction, expected, gx, gw, gb, node): (small, "
     "row_loss, dx, dw, db), or with node (loss, (small, row_loss)), the loss of that tensor class and linked to the "
     "tensors that require gradients"},
    {"bind", bind, METH_VARARGS, "bind(addresses of rh_linear_ce_workspace_bytes, rh_linear_ce, rh_scale_gradient, "
                                 "rh_last_error; workspace function; error class)"},
    {"know_unit", know_unit, METH_VARARGS, "know_unit(device, address): what lies there is 1.0 for good"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Host side of the operators.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__host(void) { return PyModule_Create(&module); }
