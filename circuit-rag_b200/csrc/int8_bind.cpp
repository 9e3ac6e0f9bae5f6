// circuit_rag._int8: the 8-bit row ops on torch tensors (CPython extension over
// the C ABI of include/circuit_ops.h; the Python face is circuit_rag/int8.py).
//
// A small call is host time: through ctypes, checks and allocations in Python
// took 10 to 13 us for a kernel of 2 us.  Here a call checks its tensors, makes
// its outputs and launches in a few microseconds.  Everything runs on the
// current stream of the tensors' device; errors come back as ValueError (a bad
// argument), RuntimeError (not a CUDA tensor, a gradient asked for) or
// circuit_rag._native.NativeLibraryError (the C entry refused or failed).
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/add.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <optional>
#include <string>

#include "../../include/circuit_ops.h"

namespace {

using at::Tensor;

struct Refused {
  PyObject* type;  // nullptr: NativeLibraryError
  std::string message;
};
[[noreturn]] void value_error(std::string m) { throw Refused{PyExc_ValueError, std::move(m)}; }
[[noreturn]] void runtime_error(std::string m) { throw Refused{PyExc_RuntimeError, std::move(m)}; }

// Lets other Python threads run: an allocation may wait for the device, and a launch behind a thousand pending ones
// waits for these.  In its scope no Python object is touched (a Refused only names its type).
struct OtherThreadsRun {
  PyThreadState* const state = PyEval_SaveThread();
  ~OtherThreadsRun() { PyEval_RestoreThread(state); }
};

PyObject* native_error() {  // borrowed: the class lives as long as its module
  PyObject* module = PyImport_ImportModule("circuit_rag._native");
  PyObject* type = module ? PyObject_GetAttrString(module, "NativeLibraryError") : nullptr;
  Py_XDECREF(module);
  if (!type) PyErr_Clear();
  return type ? type : PyExc_RuntimeError;
}

// Sets the Python error of what a call threw; nothing gets past it.
template <typename F>
PyObject* guarded(F&& f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(r.type ? r.type : native_error(), r.message.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

void native(int rc, const char* what) {
  if (!rc) return;
  const char* why = circuit_last_error();
  throw Refused{nullptr, std::string(what) + " failed (" + std::to_string(rc) + "): " + (why ? why : "")};
}

Tensor cuda_tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) runtime_error(std::string(name) + " must be CUDA tensor");
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda()) runtime_error(std::string(name) + " must be CUDA tensor");
  return t;
}
// A tensor to write.
Tensor cuda_target(PyObject* o, const char* name) {
  Tensor t = cuda_tensor(o, name);
  if (t.is_neg()) value_error(std::string(name) + " must not be a view of its negative");
  return t;
}

int type_code(at::ScalarType t) {
  return t == at::kFloat ? CIRCUIT_F32 : t == at::kHalf ? CIRCUIT_F16 : t == at::kBFloat16 ? CIRCUIT_BF16 : -1;
}
int64_t padded(int64_t dim) { return (dim + 15) / 16 * 16; }

// Elements from one row of a [n, dim] tensor to the next (a single row may carry any number).
int64_t step(const Tensor& t) {
  const int64_t s = t.stride(0), dim = t.size(1);
  return t.size(0) > 1 || s > dim ? s : dim;
}
bool plain_rows(const Tensor& t) {
  return (t.stride(1) == 1 || t.size(1) == 1) && (t.stride(0) >= t.size(1) || t.size(0) <= 1);
}
void check_dim(int64_t dim) {
  if (dim < 1 || dim > CIRCUIT_INT8_MAX_DIM)
    value_error("dim must be in [1, " + std::to_string(CIRCUIT_INT8_MAX_DIM) + "]");
}
void no_gradient(const Tensor& t, const char* name) {
  if (t.requires_grad() && at::GradMode::is_enabled())
    runtime_error(std::string(name) + " asks for a gradient: the 8-bit rows have no backward pass (use torch.no_grad())");
  // a dual tensor of forward mode, which torch.no_grad() leaves on
  if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    runtime_error(std::string(name) + " carries a forward gradient: the 8-bit rows have none (use its primal)");
}

// A tensor to read as it lies in memory: a view that stands for its negative (the imaginary part of a conjugate) as a
// copy, and one whose values do not lie next to each other (in each row).
Tensor dense(const Tensor& t) { return (t.is_neg() ? t.resolve_neg() : t).contiguous(); }
Tensor dense_rows(const Tensor& t) { return !t.is_neg() && plain_rows(t) ? t : dense(t); }

// A [n, dim] tensor of values.
Tensor value_rows(PyObject* o, const char* name) {
  Tensor t = cuda_tensor(o, name);
  if (t.dim() != 2) value_error(std::string(name) + " must have shape [n, dim]");
  if (type_code(t.scalar_type()) < 0) value_error(std::string(name) + " must be float32, float16 or bfloat16");
  no_gradient(t, name);
  check_dim(t.size(1));
  return t;
}

Tensor index_tensor(PyObject* o, const char* name, const at::Device& dev) {
  Tensor t = cuda_tensor(o, name);
  if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt)
    value_error(std::string(name) + " must be int32 or int64");
  if (t.device() != dev) value_error(std::string(name) + " must be on the rows' device");
  return t;
}

void check_pair(const Tensor& codes, const Tensor& scales, const char* name) {
  if (codes.dim() != 2 || codes.scalar_type() != at::kChar)
    value_error(std::string(name) + " codes must be int8 of shape [n, dim]");
  if (scales.dim() != 1 || scales.scalar_type() != at::kFloat || scales.size(0) != codes.size(0))
    value_error(std::string(name) + " scales must be float32 of shape [n]");
  if (scales.device() != codes.device()) value_error(std::string(name) + " codes and scales must be on one device");
  no_gradient(scales, name);
  check_dim(codes.size(1));
}
void check_target(const Tensor& t, const char* name) {
  if (!plain_rows(t)) value_error(std::string(name) + " must be contiguous in each row and its rows must not overlap");
}

// A given tensor was written: a gradient that kept it for later has to notice.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const at::Device& dev) {
  return at::detail::empty_cuda(shape, type, dev, std::nullopt);
}
// New codes [n, dim] as a view of rows padded to a multiple of 16 bytes.
Tensor fresh_codes(int64_t n, int64_t dim, const at::Device& dev) {
  Tensor t = fresh({n, padded(dim)}, at::kChar, dev);
  if (padded(dim) != dim) {
    const int64_t sizes[2] = {n, dim}, strides[2] = {padded(dim), 1};
    t.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef(sizes), at::IntArrayRef(strides));
  }
  return t;
}
// New results [nq, n]; those of 256 rows and more start their rows on 128 bytes: a warp's 32 results then fill whole
// lines (a row length off that takes the product kernel 1.7 times as long).
Tensor fresh_results(int64_t nq, int64_t n, at::ScalarType type, const at::Device& dev) {
  const int64_t line = 128 / (int64_t)c10::elementSize(type), ld = (n + line - 1) / line * line;
  if (nq < 2 || n < 256 || ld == n) return fresh({nq, n}, type, dev);
  Tensor t = fresh({nq, ld}, type, dev);
  const int64_t sizes[2] = {nq, n}, strides[2] = {ld, 1};
  t.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef(sizes), at::IntArrayRef(strides));
  return t;
}
at::ScalarType value_type(PyObject* o) {
  if (!THPDtype_Check(o)) value_error("dtype must be float32, float16 or bfloat16");
  const at::ScalarType t = reinterpret_cast<THPDtype*>(o)->scalar_type;
  if (type_code(t) < 0) value_error("dtype must be float32, float16 or bfloat16");
  return t;
}

PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* given(PyObject* o) {
  Py_INCREF(o);
  return o;
}

// quantize(rows, residual, weight, norm, eps, slots, out) -> (codes, scales, summed), or (codes, scales) without a norm
// of the root mean square.
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t count) {
  return guarded([&]() -> PyObject* {
    if (count != 7) value_error("quantize takes 7 arguments");
    Tensor rows = value_rows(a[0], "rows");
    const at::Device dev = rows.device();
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t n = rows.size(0), dim = rows.size(1);
    const long norm = PyLong_AsLong(a[3]);
    const double eps = PyFloat_AsDouble(a[4]);
    if (PyErr_Occurred()) return nullptr;
    if (!(eps >= 0.0 && eps < HUGE_VAL)) value_error("eps must be finite and not negative");
    Tensor residual, summed, weight, slots, codes, scales;
    if (a[1] != Py_None) {
      residual = value_rows(a[1], "residual");
      if (residual.sizes() != rows.sizes() || residual.scalar_type() != rows.scalar_type() || residual.device() != dev)
        value_error("residual must have the shape, type and device of rows");
    }
    if (a[2] != Py_None) {
      weight = cuda_tensor(a[2], "weight");
      if (weight.scalar_type() != rows.scalar_type() && weight.scalar_type() != at::kFloat)
        value_error("weight must be of the rows' type or float32");
      if (weight.dim() != 1 || weight.size(0) != dim || weight.device() != dev)
        value_error("weight must have shape [dim] and be on the rows' device");
      no_gradient(weight, "weight");
    }
    const bool out = a[6] != Py_None;
    if (a[5] != Py_None) {
      if (!out) value_error("slots need the store to write to as out=(codes, scales)");
      slots = index_tensor(a[5], "slots", dev);
      if (slots.dim() != 1 || slots.size(0) != n) value_error("slots must have shape [n]");
    }
    if (out) {
      if (!PyTuple_Check(a[6]) || PyTuple_GET_SIZE(a[6]) != 2) value_error("out must be a tuple (codes, scales)");
      codes = cuda_target(PyTuple_GET_ITEM(a[6], 0), "out codes");
      scales = cuda_target(PyTuple_GET_ITEM(a[6], 1), "out scales");
      check_pair(codes, scales, "out");
      check_target(codes, "out codes");
      if (!scales.is_contiguous()) value_error("out scales must be contiguous");
      if (codes.device() != dev) value_error("out must be on the rows' device");
      if (codes.size(1) != dim) value_error("out must have the rows' dim");
      if (!slots.defined() && codes.size(0) != n) value_error("out must hold as many rows as there are (or give slots)");
    }
    {
      const OtherThreadsRun scope;
      rows = dense_rows(rows);
      if (residual.defined()) residual = dense_rows(residual);
      if (weight.defined()) weight = dense(weight);
      if (slots.defined()) slots = dense(slots);
      if (!out) {
        codes = fresh_codes(n, dim, dev);
        scales = fresh({n}, at::kFloat, dev);
      }
      if (residual.defined()) summed = fresh({n, dim}, rows.scalar_type(), dev);
      if (n && codes.size(0)) {
        native(circuit_op_quantize_rows(
                   rows.const_data_ptr(), type_code(rows.scalar_type()), n, (int)dim, step(rows),
                   residual.defined() ? residual.const_data_ptr() : nullptr, residual.defined() ? step(residual) : 0,
                   weight.defined() ? weight.const_data_ptr() : nullptr,
                   weight.defined() ? type_code(weight.scalar_type()) : 0, (int)norm, (float)eps,
                   summed.defined() ? summed.mutable_data_ptr() : nullptr, dim,
                   slots.defined() ? slots.const_data_ptr() : nullptr, slots.defined() ? (int)slots.element_size() : 0,
                   codes.size(0), codes.mutable_data_ptr<int8_t>(), step(codes), scales.mutable_data_ptr<float>(),
                   c10::cuda::getCurrentCUDAStream(dev.index()).stream()),
               "quantize_rows");
        if (out) {
          written(codes);
          written(scales);
        }
      } else if (n && summed.defined()) {  // a store without rows: nothing is written, the sum is still due
        at::add_out(summed, rows, residual);
      }
    }
    PyObject* c = out ? given(PyTuple_GET_ITEM(a[6], 0)) : wrap(codes);
    PyObject* s = out ? given(PyTuple_GET_ITEM(a[6], 1)) : wrap(scales);
    if (norm != CIRCUIT_NORM_RMS) {
      PyObject* two = PyTuple_New(2);
      PyTuple_SET_ITEM(two, 0, c);
      PyTuple_SET_ITEM(two, 1, s);
      return two;
    }
    PyObject* three = PyTuple_New(3);
    PyTuple_SET_ITEM(three, 0, c);
    PyTuple_SET_ITEM(three, 1, s);
    PyTuple_SET_ITEM(three, 2, summed.defined() ? wrap(summed) : given(Py_None));
    return three;
  });
}

// dequantize(codes, scales, ids, dtype, out) -> values
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t count) {
  return guarded([&]() -> PyObject* {
    if (count != 5) value_error("dequantize takes 5 arguments");
    Tensor codes = cuda_tensor(a[0], "rows' codes"), scales = cuda_tensor(a[1], "rows' scales");
    check_pair(codes, scales, "rows'");
    const at::ScalarType type = value_type(a[3]);
    const at::Device dev = codes.device();
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t rows = codes.size(0), dim = codes.size(1);
    Tensor ids, out;
    int64_t n = rows, out_step = dim;
    if (a[2] != Py_None) {
      ids = index_tensor(a[2], "ids", dev);
      n = ids.numel();
    }
    const bool have = a[4] != Py_None;
    if (have) {
      out = cuda_target(a[4], "out");
      if (out.scalar_type() != type || out.device() != dev || out.dim() != 2 || out.size(0) != n || out.size(1) != dim)
        value_error("out must be of type dtype, of shape [" + std::to_string(n) + ", " + std::to_string(dim) +
                    "], on the rows' device");
      no_gradient(out, "out");
      check_target(out, "out");
      out_step = step(out);
    }
    {
      const OtherThreadsRun scope;
      if (!have) {
        at::DimVector shape;
        if (ids.defined()) shape.append(ids.sizes().begin(), ids.sizes().end());
        else shape.push_back(n);
        shape.push_back(dim);
        out = fresh(shape, type, dev);
      }
      codes = dense_rows(codes);
      scales = dense(scales);
      if (ids.defined()) ids = dense(ids);
      if (n)
        native(circuit_op_dequantize_rows(
                   codes.const_data_ptr<int8_t>(), step(codes), scales.const_data_ptr<float>(), rows, (int)dim,
                   ids.defined() ? ids.const_data_ptr() : nullptr, ids.defined() ? (int)ids.element_size() : 0, n,
                   out.mutable_data_ptr(), type_code(type), out_step,
                   c10::cuda::getCurrentCUDAStream(dev.index()).stream()),
               "dequantize_rows");
      if (n && have) written(out);
    }
    return have ? given(a[4]) : wrap(out);
  });
}

// Codes as the products read them: rows on 16 bytes, their padding inside the storage (a padded copy if not).
Tensor code_rows(const Tensor& codes) {
  const int64_t n = codes.size(0), dim = codes.size(1), s = step(codes), p = padded(dim);
  if (!codes.is_neg() && (dim == 1 || codes.stride(1) == 1) && s % 16 == 0 && s >= p &&
      reinterpret_cast<uintptr_t>(codes.const_data_ptr()) % 16 == 0 &&
      (p == dim || codes.storage_offset() + (n - 1) * s + p <= (int64_t)codes.storage().nbytes()))
    return codes;
  Tensor t = fresh_codes(n, dim, codes.device());
  t.copy_(codes);
  return t;
}

// scores(query_codes, query_scales, codes, scales, bias, dtype, out) -> products
PyObject* scores(PyObject*, PyObject* const* a, Py_ssize_t count) {
  return guarded([&]() -> PyObject* {
    if (count != 7) value_error("scores takes 7 arguments");
    Tensor queries = cuda_tensor(a[0], "query codes"), query_scales = cuda_tensor(a[1], "query scales");
    Tensor codes = cuda_tensor(a[2], "rows' codes"), row_scales = cuda_tensor(a[3], "rows' scales");
    check_pair(queries, query_scales, "query");
    check_pair(codes, row_scales, "rows'");
    const at::ScalarType type = value_type(a[5]);
    const at::Device dev = codes.device();
    if (queries.device() != dev) value_error("queries must be on the rows' device");
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t nq = queries.size(0), dim = queries.size(1), n = codes.size(0);
    if (codes.size(1) != dim) value_error("queries and rows must have one dim");
    if (nq > CIRCUIT_INT8_MAX_QUERIES)
      value_error("at most " + std::to_string(CIRCUIT_INT8_MAX_QUERIES) + " queries a call");
    Tensor bias, out;
    if (a[4] != Py_None) {
      bias = cuda_tensor(a[4], "bias");
      if (bias.scalar_type() != at::kFloat || bias.dim() != 1 || bias.size(0) != n || bias.device() != dev)
        value_error("bias must be float32 of shape [n] on the rows' device");
      no_gradient(bias, "bias");
    }
    int64_t out_step = n;
    const bool have = a[6] != Py_None;
    if (have) {
      out = cuda_target(a[6], "out");
      if (out.scalar_type() != type || out.device() != dev || out.dim() != 2 || out.size(0) != nq || out.size(1) != n)
        value_error("out must be of type dtype, of shape [" + std::to_string(nq) + ", " + std::to_string(n) +
                    "], on the rows' device");
      no_gradient(out, "out");
      check_target(out, "out");
      out_step = step(out);
    }
    {
      const OtherThreadsRun scope;
      if (!have) {
        out = fresh_results(nq, n, type, dev);
        out_step = step(out);
      }
      if (nq && n) {
        queries = code_rows(queries);
        codes = code_rows(codes);
        query_scales = dense(query_scales);
        row_scales = dense(row_scales);
        if (bias.defined()) bias = dense(bias);
        native(circuit_op_int8_scores(queries.const_data_ptr<int8_t>(), step(queries),
                                      query_scales.const_data_ptr<float>(), nq, codes.const_data_ptr<int8_t>(),
                                      step(codes), row_scales.const_data_ptr<float>(), n, (int)dim,
                                      bias.defined() ? bias.const_data_ptr<float>() : nullptr, out.mutable_data_ptr(),
                                      type_code(type), out_step,
                                      c10::cuda::getCurrentCUDAStream(dev.index()).stream()),
               "int8_scores");
        if (have) written(out);
      }
    }
    return have ? given(a[6]) : wrap(out);
  });
}

PyMethodDef methods[] = {
    {"quantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(quantize)), METH_FASTCALL, nullptr},
    {"dequantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dequantize)), METH_FASTCALL, nullptr},
    {"scores", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(scores)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "circuit_rag._int8", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__int8() { return PyModule_Create(&module); }
