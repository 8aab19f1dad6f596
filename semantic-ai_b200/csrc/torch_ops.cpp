// torch_ops.cpp — the operators' calls on torch tensors: checks, output tensors, the current
// stream, then the C ABI (include/svl_cuda.h), whose functions svl/_lib.py hands over at import.
//
// A step calls these several times for work of a few microseconds; made through ctypes, a call
// took 16 to 28 us on the host (three allocations, a dozen attribute reads, 19 converted
// arguments), more than the kernels themselves.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <Python.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <sstream>

#include "../../include/svl_cuda.h"

namespace {

decltype(&svl_add_norm_f8_device) g_add_norm;
decltype(&svl_f8_linear_device) g_linear;
decltype(&svl_logits_rules_device) g_rules;
decltype(&svl_last_error) g_last_error;
PyObject* g_error;  // SvlError(status, message)

constexpr int64_t kBlock = 128;

[[noreturn]] void refuse(const std::string& msg) {
  throw c10::ValueError({__func__, __FILE__, static_cast<uint32_t>(__LINE__)}, msg);
}

// A tensor argument, or null for None.
const at::Tensor* tensor(const char* name, PyObject* o, bool optional = false) {
  if (THPVariable_Check(o)) return &THPVariable_Unpack(o);
  if (optional && o == Py_None) return nullptr;
  refuse(std::string(name) + " must be a CUDA tensor");
}

std::string told(const at::Tensor& t) {
  std::ostringstream s;
  s << "got " << t.sizes() << ", " << t.scalar_type() << ", " << t.device();
  return s.str();
}

// [rows][columns] on a GPU with contiguous columns.
void check_rows(const char* name, const at::Tensor& t) {
  if (t.is_cuda() && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1)) return;
  refuse(std::string(name) + " must be a CUDA tensor [rows, columns] with contiguous columns: " + told(t));
}
void check_rows(const char* name, const at::Tensor& t, at::ScalarType type, int64_t rows, int64_t cols, c10::Device dev) {
  check_rows(name, t);
  if (t.scalar_type() == type && t.size(0) == rows && t.size(1) == cols && t.device() == dev) return;
  std::ostringstream s;
  s << name << " must be [" << rows << ", " << cols << "] of " << type << " on " << dev << ": " << told(t);
  refuse(s.str());
}
// n contiguous values; null for a tensor that is not there.
template <class T>
T* vector(const char* name, const at::Tensor* t, at::ScalarType type, int64_t n, c10::Device dev) {
  if (!t) return nullptr;
  if (t->scalar_type() == type && t->numel() == n && t->is_contiguous() && t->device() == dev)
    return static_cast<T*>(t->data_ptr());
  std::ostringstream s;
  s << name << " must be " << n << " contiguous values of " << type << " on " << dev << ": " << told(*t);
  refuse(s.str());
}

// Elements between rows (torch leaves the stride of a single row undefined).
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1)); }

int32_t dtype_of(const char* name, at::ScalarType t) {
  if (t == at::kFloat) return SVL_DT_F32;
  if (t == at::kBFloat16) return SVL_DT_BF16;
  refuse(std::string(name) + " must be float32 or bfloat16");
}

void* current_stream(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

at::Tensor empty(at::IntArrayRef size, at::ScalarType type, c10::Device dev) {
  return at::detail::empty_cuda(size, type, dev, std::nullopt);
}

// Null with the Python error set where a call failed.
bool done(svl_status status) {
  if (PyErr_Occurred()) return false;
  if (status == SVL_OK) return true;
  PyObject* e = PyObject_CallFunction(g_error, "is", (int)status, g_last_error());
  if (e) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
  return false;
}

bool count(Py_ssize_t got, Py_ssize_t want) {
  if (got == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments wanted, %zd given", want, got);
  return false;
}

// x, residual, norm kind, weight, bias, eps, out_sum -> (q, scales, h)
PyObject* add_norm_f8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!count(n, 7)) return nullptr;
  const at::Tensor& x = *tensor("x", a[0]);
  check_rows("x", x);
  const int64_t rows = x.size(0), k = x.size(1), ld = (k + 15) / 16 * 16;
  const c10::Device dev = x.device();
  const at::ScalarType type = x.scalar_type();
  const int32_t dtype = dtype_of("x", type);
  const at::Tensor* residual = tensor("residual", a[1], true);
  if (residual) check_rows("residual", *residual, type, rows, k, dev);
  const long kind = PyLong_AsLong(a[2]);
  const double eps = PyFloat_AsDouble(a[5]);
  if (PyErr_Occurred()) return nullptr;
  const float* w = vector<float>("weight", tensor("weight", a[3], true), at::kFloat, k, dev);
  const float* b = vector<float>("bias", tensor("bias", a[4], true), at::kFloat, k, dev);
  const at::Tensor* given = tensor("out_sum", a[6], true);
  if (given) check_rows("out_sum", *given, type, rows, k, dev);
  const at::Tensor h = given ? *given : residual ? empty({rows, k}, type, dev) : x;
  const bool keep = given || residual;
  at::Tensor q = ld == k ? empty({rows, k}, at::kFloat8_e4m3fn, dev)
                         : at::detail::empty_strided_cuda({rows, k}, {ld, 1}, at::kFloat8_e4m3fn, dev);
  at::Tensor scales = empty({(k + kBlock - 1) / kBlock, rows}, at::kFloat, dev);
  const svl_status s = g_add_norm(dev.index(), rows, (int32_t)std::min<int64_t>(k, INT32_MAX), dtype, x.data_ptr(),
                                  row_stride(x), residual ? residual->data_ptr() : nullptr,
                                  residual ? row_stride(*residual) : 0, (int32_t)kind, w, b, (float)eps,
                                  keep ? h.data_ptr() : nullptr, row_stride(h), static_cast<uint8_t*>(q.data_ptr()), ld,
                                  static_cast<float*>(scales.data_ptr()), rows, current_stream(dev));
  if (!done(s)) return nullptr;
  PyObject* out = PyTuple_New(3);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(q)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(scales)));
  if (given || !residual) {
    PyObject* same = given ? a[6] : a[0];
    Py_INCREF(same);
    PyTuple_SET_ITEM(out, 2, same);
  } else {
    PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(h));
  }
  return out;
  END_HANDLE_TH_ERRORS
}

// handle, n, k, device index, q, scales, out dtype, out -> out
PyObject* f8_linear(PyObject*, PyObject* const* a, Py_ssize_t cnt) {
  HANDLE_TH_ERRORS
  if (!count(cnt, 8)) return nullptr;
  void* handle = PyLong_AsVoidPtr(a[0]);
  const long n = PyLong_AsLong(a[1]), k = PyLong_AsLong(a[2]), index = PyLong_AsLong(a[3]);
  if (PyErr_Occurred()) return nullptr;
  const c10::Device dev(c10::kCUDA, (c10::DeviceIndex)index);
  const at::Tensor &q = *tensor("q", a[4]), &scales = *tensor("scales", a[5]);
  check_rows("q", q);
  const int64_t rows = q.size(0);
  check_rows("q", q, at::kFloat8_e4m3fn, rows, k, dev);
  check_rows("scales", scales, at::kFloat, (k + kBlock - 1) / kBlock, rows, dev);
  const at::Tensor* given = tensor("out", a[7], true);
  if (!given && !THPDtype_Check(a[6])) refuse("out_dtype must be a torch.dtype");
  const at::ScalarType type = given ? given->scalar_type() : reinterpret_cast<THPDtype*>(a[6])->scalar_type;
  const int32_t dtype = dtype_of(given ? "out" : "out_dtype", type);
  if (given) check_rows("out", *given, type, rows, n, dev);
  at::Tensor out = given ? *given : empty({rows, n}, type, dev);
  // A single row's stride is never used.
  const int64_t ld = rows > 1 ? q.stride(0) : (k + 15) / 16 * 16;
  const svl_status s = g_linear(static_cast<svl_f8_linear*>(handle), rows, static_cast<const uint8_t*>(q.data_ptr()), ld,
                                static_cast<const float*>(scales.data_ptr()), row_stride(scales), dtype, out.data_ptr(),
                                row_stride(out), current_stream(dev));
  if (!done(s)) return nullptr;
  if (given) {
    Py_INCREF(a[7]);
    return a[7];
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// logits, history, lengths, repetition, frequency, presence, dense_bias, bias_ids, bias_values,
// masks, mask_rows, first_penalised, append, out -> (logits, tokens)
PyObject* logits_rules(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!count(n, 14)) return nullptr;
  const at::Tensor& logits = *tensor("logits", a[0]);
  check_rows("logits", logits);
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  const c10::Device dev = logits.device();
  const at::ScalarType type = logits.scalar_type();
  const int32_t dtype = dtype_of("logits", type);
  svl_logits_rules r{};
  const long first = PyLong_AsLong(a[11]);
  const int append = PyObject_IsTrue(a[12]);
  if (PyErr_Occurred()) return nullptr;
  if (first < 0 || first > INT32_MAX) refuse("first_penalised must be a token id");
  r.first_penalised = (int32_t)first;
  const at::Tensor *history = tensor("history", a[1], true), *lengths = tensor("lengths", a[2], true);
  if (!history != !lengths) refuse("history and lengths go together");
  if (history) {
    check_rows("history", *history);
    check_rows("history", *history, at::kInt, rows, history->size(1), dev);
    int32_t* len = vector<int32_t>("lengths", lengths, at::kInt, rows, dev);
    if (history->size(1)) {
      r.d_history = static_cast<int32_t*>(history->data_ptr());
      r.history_stride = row_stride(*history);
      r.history_cap = (int32_t)std::min<int64_t>(history->size(1), INT32_MAX);
      r.d_lengths = len;
    }
  }
  r.d_repetition = vector<float>("repetition", tensor("repetition", a[3], true), at::kFloat, rows, dev);
  r.d_frequency = vector<float>("frequency", tensor("frequency", a[4], true), at::kFloat, rows, dev);
  r.d_presence = vector<float>("presence", tensor("presence", a[5], true), at::kFloat, rows, dev);
  r.d_dense_bias = vector<float>("dense_bias", tensor("dense_bias", a[6], true), at::kFloat, vocab, dev);
  const at::Tensor *ids = tensor("bias_ids", a[7], true), *values = tensor("bias_values", a[8], true);
  if (!ids != !values) refuse("bias_ids and bias_values go together");
  if (ids) {
    check_rows("bias_ids", *ids);
    check_rows("bias_ids", *ids, at::kInt, rows, ids->size(1), dev);
    check_rows("bias_values", *values, at::kFloat, rows, ids->size(1), dev);
    if (rows > 1 && ids->stride(0) != values->stride(0)) refuse("bias_ids and bias_values must have the same row stride");
    if (ids->size(1)) {
      r.d_bias_ids = static_cast<const int32_t*>(ids->data_ptr());
      r.d_bias_values = static_cast<const float*>(values->data_ptr());
      r.bias_stride = row_stride(*ids);
      r.bias_cap = (int32_t)std::min<int64_t>(ids->size(1), INT32_MAX);
    }
  }
  if (const at::Tensor* masks = tensor("masks", a[9], true)) {
    check_rows("masks", *masks);
    check_rows("masks", *masks, at::kInt, masks->size(0), std::max(masks->size(1), (vocab + 31) / 32), dev);
    if (masks->size(0)) {
      r.d_masks = static_cast<const uint32_t*>(masks->data_ptr());
      r.mask_stride = row_stride(*masks);
      r.n_masks = (int32_t)masks->size(0);
    }
  }
  r.d_mask_rows = vector<int32_t>("mask_rows", tensor("mask_rows", a[10], true), at::kInt, rows, dev);
  r.append = append;
  const at::Tensor* given = tensor("out", a[13], true);
  if (given) check_rows("out", *given, type, rows, vocab, dev);
  at::Tensor out = given ? *given : empty({rows, vocab}, type, dev);
  at::Tensor tokens = empty({rows}, at::kInt, dev);
  const svl_status s = g_rules(dev.index(), rows, (int32_t)std::min<int64_t>(vocab, INT32_MAX), dtype, logits.data_ptr(),
                               row_stride(logits), &r, out.data_ptr(), row_stride(out),
                               static_cast<int32_t*>(tokens.data_ptr()), current_stream(dev));
  if (!done(s)) return nullptr;
  PyObject* both = PyTuple_New(2);
  if (!both) return nullptr;
  if (given) Py_INCREF(a[13]);
  PyTuple_SET_ITEM(both, 0, given ? a[13] : THPVariable_Wrap(std::move(out)));
  PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(tokens)));
  return both;
  END_HANDLE_TH_ERRORS
}

// Addresses of the four C functions, and the class of their errors.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count(n, 5)) return nullptr;
  g_add_norm = reinterpret_cast<decltype(g_add_norm)>(PyLong_AsVoidPtr(a[0]));
  g_linear = reinterpret_cast<decltype(g_linear)>(PyLong_AsVoidPtr(a[1]));
  g_rules = reinterpret_cast<decltype(g_rules)>(PyLong_AsVoidPtr(a[2]));
  g_last_error = reinterpret_cast<decltype(g_last_error)>(PyLong_AsVoidPtr(a[3]));
  if (PyErr_Occurred()) return nullptr;
  Py_INCREF(a[4]);
  Py_XDECREF(g_error);
  g_error = a[4];
  Py_RETURN_NONE;
}

#define METHOD(name) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr }
PyMethodDef g_methods[] = {METHOD(bind), METHOD(add_norm_f8), METHOD(f8_linear), METHOD(logits_rules),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&g_module); }
