// Native host side of the operators on rows in 8 bits (include/hstu_rows8.h): a call of recml_amd.Rows8, quantize_rows, norm_rows8,
// Rows8.values or gemm_rows8 goes through ONE function here to the kernels.
//
// What a function here does not take as it is (a conversion, a copy, an error to report) comes back as None, and the Python side
// (recml_amd/hstu_rows8.py), which knows every form and every message, runs.

#include "native_common.h"

#include <torch/csrc/Dtype.h>

#include <limits>
#include <utility>

#include "hstu_rows8.h"

namespace {

// What the Python side raises for these: arguments that are refused are a ValueError.
void rows8_check(int rc, const char* what) {
  TORCH_CHECK_VALUE(rc != HSTU_ROWS8_ERR_NULL && rc != HSTU_ROWS8_ERR_SHAPE, what, " rejected the arguments (", rc, "): ", hstu_rows8_last_error());
  TORCH_CHECK(rc == HSTU_ROWS8_OK, what, " failed (", rc, "): ", hstu_rows8_last_error());
}

constexpr int64_t MOST = std::numeric_limits<int32_t>::max();

template <typename A>
void head(A* a) {
  memset(a, 0, sizeof(*a));
  a->struct_size = sizeof(*a);
  a->version = HSTU_ROWS8_ABI_VERSION;
}

bool fill(const Tensor& codes, const Tensor& exponents, int64_t width, HstuRows8* r) {
  if (!codes.defined() || !exponents.defined() || !codes.is_cuda() || width < 1 || width > HSTU_ROWS8_MAX_WIDTH) return false;
  const auto dev = codes.device();
  if (!plain(codes, dev, at::kByte) || !plain(exponents, dev, at::kByte) || codes.dim() != 2 || exponents.dim() != 3 || codes.size(0) > MOST) return false;
  const int64_t blocks = (width + 127) / 128;
  if (codes.size(1) != 128 * blocks || exponents.size(0) != (blocks + 3) / 4 || exponents.size(1) != codes.size(0) || exponents.size(2) != 4) return false;
  if (!aligned(codes) || ((uintptr_t)exponents.const_data_ptr() & 3u)) return false;
  r->codes = const_cast<void*>(codes.const_data_ptr());
  r->exponents = const_cast<void*>(exponents.const_data_ptr());
  r->rows = codes.size(0);
  r->width = (int32_t)width;
  return true;
}

bool dtype_arg(PyObject* o, at::ScalarType* out) {
  if (!THPDtype_Check(o)) return false;
  *out = ((THPDtype*)o)->scalar_type;
  return *out == at::kFloat || *out == at::kBFloat16;
}

int32_t dtype_of(at::ScalarType t) { return t == at::kFloat ? HSTU_ROWS8_FP32 : HSTU_ROWS8_BF16; }

// [..., W] whose leading axes collapse to one row stride.
bool flat(const Tensor& t, int64_t* stride) {
  const int64_t n = t.dim();
  if (n < 1 || (t.size(n - 1) > 1 && t.stride(n - 1) != 1)) return false;
  *stride = 0;
  int64_t next = -1;                 // stride times size of the axes behind
  for (int64_t i = n - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (next < 0) *stride = t.stride(i);
    else if (t.stride(i) != next) return false;
    next = t.stride(i) * t.size(i);
  }
  return true;
}

// New codes and exponents: one allocation, and tensors over its two parts (an allocation is a fifth of a small call's host time).
void fresh_rows(const Tensor& like, int64_t rows, int64_t width, Tensor* codes, Tensor* exponents) {
  const int64_t blocks = (width + 127) / 128, bytes = rows * 128 * blocks;
  const Tensor all = at::empty({bytes + (blocks + 3) / 4 * rows * 4}, like.options().dtype(at::kByte).requires_grad(false));
  auto part = [&](int64_t from, at::IntArrayRef sizes) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(from);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    return t;
  };
  *codes = part(0, {rows, 128 * blocks});
  *exponents = part(bytes, {(blocks + 3) / 4, rows, 4});
}

// check_rows8(codes, exponents, width): whether they are rows in 8 bits.
PyObject* check_rows8(PyObject*, PyObject* const* a, Py_ssize_t count) {
  if (count != 3) {
    PyErr_SetString(PyExc_TypeError, "check_rows8 takes 3 arguments");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    if (!THPVariable_Check(a[0]) || !THPVariable_Check(a[1])) Py_RETURN_FALSE;
    HstuRows8 r;
    int64_t width;
    return PyBool_FromLong(long_arg(a[2], &width) && fill(THPVariable_Unpack(a[0]), THPVariable_Unpack(a[1]), width, &r));
  });
}

// norm_rows8(x, gamma, beta, eps, gate, add, kind) -> (codes, exponents, width, sum or None), or None
PyObject* norm_rows8(PyObject*, PyObject* const* a, Py_ssize_t count) {
  if (count != 7) {
    PyErr_SetString(PyExc_TypeError, "norm_rows8 takes 7 arguments");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Tensor x, gamma, beta, gate, add, codes, exponents, sum;
    HstuRows8NormArgs args;
    head(&args);
    double eps;
    int64_t kind;
    if (!tensor_arg(a[0], &x) || !tensor_arg(a[1], &gamma) || !tensor_arg(a[2], &beta) || !float_arg(a[3], &eps) || !tensor_arg(a[4], &gate) ||
        !tensor_arg(a[5], &add) || !long_arg(a[6], &kind)) Py_RETURN_NONE;
    if (!x.defined() || !x.is_cuda() || (x.scalar_type() != at::kFloat && x.scalar_type() != at::kBFloat16) || !flat(x, &args.x_stride)) Py_RETURN_NONE;
    const auto dev = x.device();
    const auto type = x.scalar_type();
    const int64_t W = x.size(x.dim() - 1);
    if (W < 1 || W > HSTU_ROWS8_MAX_WIDTH || x.numel() / W > MOST) Py_RETURN_NONE;
    for (const Tensor* t : {&gamma, &beta})
      if (t->defined() && (!plain(*t, dev, type) || t->numel() != W)) Py_RETURN_NONE;
    if (kind != HSTU_ROWS8_AS_IS && !gamma.defined()) Py_RETURN_NONE;
    if (gate.defined() && (!on(gate, dev) || gate.scalar_type() != type || gate.sizes() != x.sizes() || !flat(gate, &args.gate_stride))) Py_RETURN_NONE;
    if (add.defined() && (!on(add, dev) || add.scalar_type() != type || add.sizes() != x.sizes() || !flat(add, &args.add_stride))) Py_RETURN_NONE;
    if (wants_grad({&x, &gamma, &beta, &gate, &add}) || dual({&x, &gamma, &beta, &gate, &add})) Py_RETURN_NONE;
    without_lock(x, [&] {
      const int64_t R = x.numel() / W;
      fresh_rows(x, R, W, &codes, &exponents);
      if (add.defined()) sum = at::empty(x.sizes(), x.options().requires_grad(false));
      args.rows.codes = codes.data_ptr(); args.rows.exponents = exponents.data_ptr();
      args.rows.rows = R; args.rows.width = (int32_t)W;
      args.norm = (int32_t)kind; args.dtype = dtype_of(type); args.eps = (float)eps;
      auto at_ = [](const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; };
      args.x = at_(x); args.gamma = at_(gamma); args.beta = at_(beta); args.gate = at_(gate); args.add = at_(add);
      if (sum.defined()) { args.sum = sum.data_ptr(); args.sum_stride = W; }
      rows8_check(hstu_rows8_norm(&args, stream_of(x)), "hstu_rows8_norm");
      return true;
    });
    if (sum.defined()) return Py_BuildValue("(NNLN)", THPVariable_Wrap(std::move(codes)), THPVariable_Wrap(std::move(exponents)), (long long)W, THPVariable_Wrap(std::move(sum)));
    return Py_BuildValue("(NNLO)", THPVariable_Wrap(std::move(codes)), THPVariable_Wrap(std::move(exponents)), (long long)W, Py_None);
  });
}

// read_rows8(codes, exponents, width, dtype) -> Tensor, or None
PyObject* read_rows8(PyObject*, PyObject* const* a, Py_ssize_t count) {
  if (count != 4) {
    PyErr_SetString(PyExc_TypeError, "read_rows8 takes 4 arguments");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Tensor codes, exponents, out;
    HstuRows8ReadArgs args;
    head(&args);
    int64_t width;
    at::ScalarType type;
    if (!tensor_arg(a[0], &codes) || !tensor_arg(a[1], &exponents) || !long_arg(a[2], &width) || !dtype_arg(a[3], &type) ||
        !fill(codes, exponents, width, &args.rows)) Py_RETURN_NONE;
    without_lock(codes, [&] {
      out = at::empty({codes.size(0), width}, codes.options().dtype(type));
      args.out = out.data_ptr(); args.out_stride = width; args.dtype = dtype_of(type);
      rows8_check(hstu_rows8_read(&args, stream_of(codes)), "hstu_rows8_read");
      return true;
    });
    return THPVariable_Wrap(std::move(out));
  });
}

// gemm_rows8(x_codes, x_exponents, w_codes, w_exponents, width, bias, activation, residual, dtype) -> Tensor, or None
PyObject* gemm_rows8(PyObject*, PyObject* const* a, Py_ssize_t count) {
  if (count != 9) {
    PyErr_SetString(PyExc_TypeError, "gemm_rows8 takes 9 arguments");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Tensor x, xe, w, we, bias, residual, out;
    HstuRows8GemmArgs args;
    head(&args);
    int64_t width;
    at::ScalarType type;
    if (!tensor_arg(a[0], &x) || !tensor_arg(a[1], &xe) || !tensor_arg(a[2], &w) || !tensor_arg(a[3], &we) || !long_arg(a[4], &width) ||
        !tensor_arg(a[5], &bias) || !PyBool_Check(a[6]) || !tensor_arg(a[7], &residual) || !dtype_arg(a[8], &type)) Py_RETURN_NONE;
    if (!fill(x, xe, width, &args.x) || !fill(w, we, width, &args.w) || x.device() != w.device()) Py_RETURN_NONE;
    const auto dev = x.device();
    const int64_t M = x.size(0), N = w.size(0);
    if (bias.defined() && (!plain(bias, dev, type) || bias.numel() != N)) Py_RETURN_NONE;
    if (residual.defined()) {
      if (!on(residual, dev) || residual.scalar_type() != type || residual.dim() != 2 || residual.size(0) != M || residual.size(1) != N ||
          !flat(residual, &args.c_stride)) Py_RETURN_NONE;
      args.c = residual.const_data_ptr();
    }
    if (wants_grad({&bias, &residual}) || dual({&bias, &residual})) Py_RETURN_NONE;
    if (bias.defined()) args.bias = bias.const_data_ptr();
    args.activation = a[6] == Py_True ? 1 : 0;
    args.dtype = dtype_of(type);
    without_lock(x, [&] {
      out = at::empty({M, N}, x.options().dtype(type));
      args.out = out.data_ptr(); args.out_stride = N;
      rows8_check(hstu_rows8_gemm(&args, stream_of(x)), "hstu_rows8_gemm");
      return true;
    });
    return THPVariable_Wrap(std::move(out));
  });
}

PyMethodDef methods[] = {
#define HSTU_FAST(name, doc) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, doc}
    HSTU_FAST(check_rows8, "Whether tensors are rows in 8 bits."),
    HSTU_FAST(norm_rows8, "Rows, normed or as they are, into 8 bits."),
    HSTU_FAST(read_rows8, "What rows in 8 bits stand for."),
    HSTU_FAST(gemm_rows8, "The product of rows in 8 bits."),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native_rows8", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native_rows8(void) { return PyModule_Create(&module); }
