// What the native host sides (native.cpp, native_serve.cpp) share: arguments from Python, and how a call runs.

#ifndef RECML_AMD_NATIVE_COMMON_H_
#define RECML_AMD_NATIVE_COMMON_H_

#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <hip/hip_runtime.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/edge.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/grad_mode.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <initializer_list>

namespace {

using at::Tensor;

void* stream_of(const Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

bool capturing(void* stream) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing((hipStream_t)stream, &st) == hipSuccess && st != hipStreamCaptureStatusNone;
}

// An optional tensor argument: false when it is something that the Python side has to look at.
bool tensor_arg(PyObject* o, Tensor* out) {
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  *out = THPVariable_Unpack(o);
  return true;
}

bool float_arg(PyObject* o, double* out) {
  if (PyFloat_CheckExact(o)) { *out = PyFloat_AS_DOUBLE(o); return true; }
  if (PyLong_CheckExact(o)) {
    *out = PyLong_AsDouble(o);
    if (*out == -1.0 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    return true;
  }
  return false;
}

bool long_arg(PyObject* o, int64_t* out) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *out = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow == 0;
}

bool on(const Tensor& t, c10::Device dev) { return t.is_cuda() && t.device() == dev; }

bool plain(const Tensor& t, c10::Device dev, at::ScalarType type) { return on(t, dev) && t.scalar_type() == type && t.is_contiguous(); }

// fp32 [heads, width] or [width] table with heads in {1, H}
bool table(const Tensor& t, c10::Device dev, int64_t H, int64_t* heads, int64_t* width) {
  if (!plain(t, dev, at::kFloat) || t.dim() < 1 || t.dim() > 2) return false;
  *heads = t.dim() == 2 ? t.size(0) : 1;
  *width = t.size(t.dim() - 1);
  return *heads == 1 || *heads == H;
}

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Whether a tensor carries a forward-mode tangent.  The kernels give none for their results: such a call goes the Python way, whose
// torch steps carry tangents on and whose autograd functions refuse them.
bool dual(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined()) return true;
  return false;
}

bool aligned(const Tensor& t) { return ((uintptr_t)t.const_data_ptr() & 15u) == 0; }

Tensor fresh(const Tensor& like, at::IntArrayRef shape) { return at::empty(shape, like.options().requires_grad(false)); }

// A tensor kept for the backward, the forward's own intermediates included: this way torch's saved-tensor hooks see it (checkpointing
// and offloading replace it).
torch::autograd::SavedVariable keep(const Tensor& t) { return torch::autograd::SavedVariable(t, false); }

// Runs `f`; an exception becomes the Python one of its type (torch.OutOfMemoryError, IndexError, an error of a hook, ...).
template <typename F>
PyObject* guarded(F&& f) {
  HANDLE_TH_ERRORS
  return f();
  END_HANDLE_TH_ERRORS
}

// Runs `f` without the interpreter's lock, on the tensor's device, outside of any graph.
template <typename F>
auto without_lock(const Tensor& t, F&& f) {
  struct Release {
    PyThreadState* saved = PyEval_SaveThread();
    ~Release() { PyEval_RestoreThread(saved); }
  } release;
  const c10::DeviceGuard guard(t.device());
  const at::NoGradGuard no_grad;
  return f();
}

}  // namespace

#endif  // RECML_AMD_NATIVE_COMMON_H_
