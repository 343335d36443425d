// Python binding of the gradient norm (module muon_sr_b200._native): reads the tensors' fields,
// allocates the results and calls the C ABI in one call from Python. Reading a few hundred
// tensors attribute by attribute in Python takes longer than their norm on the GPU.
//
// It serves plain gradients only: strided, contiguous CUDA tensors of one device and of the
// supported types, each once. For anything else a function returns None without having done
// anything, and the caller goes through kernels.GradTable, which copies or refuses.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <vector>

#include "../../include/muon_sr_b200.h"

namespace {

struct Gradients {
  std::vector<msr_grad_entry> entries;
  std::vector<c10::TensorImpl*> tensors;  // alive as long as the list they came from
  int device = -1;
};

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return MSR_BF16;
    case at::kHalf: return MSR_FP16;
    case at::kFloat: return MSR_FP32;
    default: return -1;
  }
}

// The entries of the tensors in `list` (of their .grad with `of_grads`, those without one left
// out); false where one is not plain.
bool collect(PyObject* list, bool of_grads, Gradients& out) {
  if (!PyList_CheckExact(list)) return false;
  const Py_ssize_t n = PyList_GET_SIZE(list);
  out.entries.reserve(n);
  out.tensors.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* item = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(item)) return false;
    const at::Tensor& t = THPVariable_Unpack(item);
    if (of_grads && !t.is_leaf()) return false;  // (Python warns about .grad of such a tensor)
    const at::Tensor& g = of_grads ? t.grad() : t;
    if (!g.defined()) {
      if (of_grads) continue;
      return false;
    }
    if (g.layout() != at::kStrided || !g.is_cuda() || g.unsafeGetTensorImpl()->is_python_dispatch() ||
        !g.is_contiguous())
      return false;
    const int code = dtype_code(g.scalar_type());
    const int device = g.get_device();
    if (code < 0 || (out.device >= 0 && device != out.device)) return false;
    out.device = device;
    out.tensors.push_back(g.unsafeGetTensorImpl());
    out.entries.push_back(msr_grad_entry{g.numel() ? g.data_ptr() : nullptr, g.numel(), code, 0});
  }
  return !out.entries.empty();
}

// Whether two entries start at the same place (the same gradient twice).
bool repeated(const Gradients& g) {
  std::vector<const void*> p;
  p.reserve(g.entries.size());
  for (const msr_grad_entry& e : g.entries)
    if (e.numel > 0) p.push_back(e.grad);
  std::sort(p.begin(), p.end());
  return std::adjacent_find(p.begin(), p.end()) != p.end();
}

void check(int status, const char* what) {
  if (status != MSR_OK)
    throw std::runtime_error(std::string(what) + " failed: " + msr_status_string(status) + ": " + msr_last_error());
}

// The memory of one call, on the gradients' device and its current stream.
struct Call {
  c10::cuda::CUDAGuard guard;
  at::Tensor state, workspace;
  size_t bytes;
  msr_stream_t stream;

  explicit Call(const Gradients& g) : guard(static_cast<c10::DeviceIndex>(g.device)) {
    const at::TensorOptions on = at::TensorOptions().device(at::kCUDA, g.device);
    bytes = msr_grad_norm_workspace_bytes(static_cast<int>(g.entries.size()));
    state = at::empty({static_cast<int64_t>(sizeof(msr_clip_state) / 4)}, on.dtype(at::kFloat));
    workspace = at::empty({static_cast<int64_t>(bytes)}, on.dtype(at::kByte));
    stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(g.device)).stream();
  }
  msr_clip_state* st() { return reinterpret_cast<msr_clip_state*>(state.data_ptr()); }
  at::Tensor norm() { return state.select(0, offsetof(msr_clip_state, norm) / 4); }
};

// grad_norm(list, norm, scale, max_norm, per_tensor, of_grads) -> (state, norm, each or None), or None
PyObject* grad_norm(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject* list;
  int norm, per_tensor, of_grads;
  double scale, max_norm;
  if (!PyArg_ParseTuple(args, "Oiddpp", &list, &norm, &scale, &max_norm, &per_tensor, &of_grads)) return nullptr;
  Gradients g;
  if (!collect(list, of_grads, g) || (of_grads && repeated(g))) Py_RETURN_NONE;
  const at::AutoDispatchBelowADInplaceOrView plain;
  Call call(g);
  const int count = static_cast<int>(g.entries.size());
  at::Tensor each;
  if (per_tensor) each = at::empty({count}, call.state.options());
  check(msr_grad_norm(g.entries.data(), count, norm, scale, max_norm, call.st(),
                      per_tensor ? each.data_ptr<float>() : nullptr, call.workspace.data_ptr(), call.bytes, call.stream),
        "msr_grad_norm");
  if (per_tensor)
    return Py_BuildValue("NNN", THPVariable_Wrap(call.state), THPVariable_Wrap(call.norm()), THPVariable_Wrap(each));
  return Py_BuildValue("NNO", THPVariable_Wrap(call.state), THPVariable_Wrap(call.norm()), Py_None);
  END_HANDLE_TH_ERRORS
}

// grad_clip(parameters, norm, scale, max_norm) -> norm, or None
PyObject* grad_clip(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  PyObject* list;
  int norm;
  double scale, max_norm;
  if (!PyArg_ParseTuple(args, "Oidd", &list, &norm, &scale, &max_norm)) return nullptr;
  Gradients g;
  if (!collect(list, true, g) || repeated(g)) Py_RETURN_NONE;
  const at::AutoDispatchBelowADInplaceOrView plain;
  Call call(g);
  check(msr_grad_clip(g.entries.data(), static_cast<int>(g.entries.size()), norm, scale, max_norm, call.st(),
                      call.workspace.data_ptr(), call.bytes, call.stream),
        "msr_grad_clip");
  for (c10::TensorImpl* t : g.tensors)  // autograd sees the write, as after any in-place operation
    if (!t->is_inference()) t->bump_version();
  return THPVariable_Wrap(call.norm());
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"grad_norm", grad_norm, METH_VARARGS, nullptr},
    {"grad_clip", grad_clip, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// `built_for` names the torch and interpreter of the build; _lib.native() refuses any other.
PyMODINIT_FUNC PyInit__native() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", MSR_BUILT_FOR) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
