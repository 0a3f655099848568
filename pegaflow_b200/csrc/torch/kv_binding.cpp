// The paged-cache operators for torch tensors (pegaflow_b200/kv.py): argument
// checks, new tensors, the stream, one call into the library each. In C++ because
// a decode step's calls run for a few microseconds: the same in Python took longer
// than the kernels.
//
// Checks raise ValueError; the library's own become PegaError by _native.check.
// Everything that a call works on is in its arguments: nothing is kept.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <exception>
#include <optional>
#include <sstream>
#include <string>

#include "pegaflow.h"

namespace {

struct ValueError : std::exception {
  std::string text;
  explicit ValueError(std::string t) : text(std::move(t)) {}
  const char* what() const noexcept override { return text.c_str(); }
};
struct PythonError {};  // one is set

[[noreturn]] void refuse(const std::string& text) { throw ValueError(text); }

template <typename T>
std::string shown(at::ArrayRef<T> v) {
  std::ostringstream s;
  s << "[";
  for (size_t i = 0; i < v.size(); ++i) s << (i ? ", " : "") << v[i];
  s << "]";
  return s.str();
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) refuse(std::string(what) + " must be a tensor");
  return THPVariable_Unpack(o);
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PythonError();
  return v;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PythonError();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PythonError();
  return v;
}

std::optional<uint32_t> rows_dtype(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return PF_DTYPE_BF16;
    case at::kHalf: return PF_DTYPE_FP16;
    case at::kFloat: return PF_DTYPE_FP32;
    default: return std::nullopt;
  }
}

// A KVCache's description, and the device that it is on (-1: the CPU).
struct Cache {
  const pf_kv_cache* c;
  int index;
  std::string on() const { return index < 0 ? "cpu" : "cuda:" + std::to_string(index); }
  void need_cuda() const {
    if (index < 0) refuse("the cache must be on a CUDA device");
  }
};
Cache cache(PyObject* address, PyObject* index) {
  return Cache{reinterpret_cast<const pf_kv_cache*>(static_cast<uintptr_t>(integer(address))), int(integer(index))};
}

// The operators have no backward pass: a result or a cache without it would stop the gradient and say nothing.
void need_no_gradient(const at::Tensor& t, const char* what) {
  if (t.requires_grad() && c10::GradMode::is_enabled()) {
    refuse(std::string(what) + " requires a gradient, which these operators do not compute: call them under torch.no_grad(), or detach it");
  }
}

pf_kv_rows rows(const Cache& c, const at::Tensor& t, int64_t n, int64_t heads, const char* what) {
  const int64_t dim = c.c->head_dim;
  if (t.dim() != 3 || t.size(0) != n || t.size(1) != heads || t.size(2) != dim || t.get_device() != c.index ||
      (dim > 1 && t.stride(2) != 1)) {
    std::ostringstream s;
    s << what << " must be [" << n << ", " << heads << ", " << dim << "] with a contiguous last axis on " << c.on() << ", not "
      << shown(t.sizes()) << " with strides " << shown(t.strides()) << " on " << t.device();
    refuse(s.str());
  }
  need_no_gradient(t, what);
  return pf_kv_rows{reinterpret_cast<uint64_t>(t.data_ptr()), t.stride(0), t.stride(1)};
}

const at::Tensor& ints(const Cache& c, PyObject* o, at::ScalarType dtype, int64_t dim, const char* what) {
  const at::Tensor& t = tensor(o, what);
  if (t.scalar_type() != dtype || t.dim() != dim || t.get_device() != c.index || (t.size(dim - 1) > 1 && t.stride(dim - 1) != 1)) {
    refuse(std::string(what) + " must be " + (dtype == at::kLong ? "int64" : "int32") + " with " + std::to_string(dim) +
           " axes, the last contiguous, on " + c.on());
  }
  return t;
}

int32_t* status_of(const Cache& c, PyObject* o) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, "status");
  if (t.scalar_type() != at::kInt || t.numel() != 1 || t.get_device() != c.index) refuse("status must be one int32 on " + c.on());
  return t.data_ptr<int32_t>();
}

// The stream of a call, current while it makes new tensors: they belong to it.
struct Stream {
  c10::cuda::OptionalCUDAStreamGuard guard;
  cudaStream_t raw;
  Stream(const Cache& c, PyObject* given) {
    c.need_cuda();
    if (given == Py_None) {
      raw = c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(c.index)).stream();
    } else {
      raw = reinterpret_cast<cudaStream_t>(static_cast<uintptr_t>(integer(given)));
      guard.reset_stream(c10::cuda::getStreamFromExternal(raw, c10::DeviceIndex(c.index)));
    }
  }
};

at::Tensor made(const Cache& c, at::IntArrayRef shape, at::ScalarType dtype) {
  return at::empty(shape, at::TensorOptions().dtype(dtype).device(at::kCUDA, c10::DeviceIndex(c.index)));
}

void check(int rc) {
  if (rc == PF_OK) return;
  PyObject* native = PyImport_ImportModule("pegaflow_b200._native");
  PyObject* done = native ? PyObject_CallMethod(native, "check", "i", rc) : nullptr;
  Py_XDECREF(native);
  Py_XDECREF(done);
  if (done) PyErr_SetString(PyExc_RuntimeError, pf_last_error());
  throw PythonError();
}

// Runs f with what it throws as a Python error.
template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F&& f) {
  try {
    if (got != want) refuse("wrong number of arguments");
    return f();
  } catch (const ValueError& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const PythonError&) {
  } catch (const std::bad_alloc&) {
    PyErr_NoMemory();
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// write(cache, index, key, value, slots, given_scales, status, stream)
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t count) {
  return guarded(count, 8, [&]() -> PyObject* {
    const Cache c = cache(a[0], a[1]);
    const at::Tensor &key = tensor(a[2], "key"), &value = tensor(a[3], "value");
    const auto dtype = rows_dtype(key.scalar_type());
    if (!dtype || value.scalar_type() != key.scalar_type()) {
      refuse(std::string("key and value must both be bfloat16, float16 or float32, not ") + at::toString(key.scalar_type()) + " and " +
             at::toString(value.scalar_type()));
    }
    const int64_t n = key.dim() ? key.size(0) : 0;
    const pf_kv_rows k = rows(c, key, n, c.c->heads, "key"), v = rows(c, value, n, c.c->heads, "value");
    const at::Tensor& slots = ints(c, a[4], at::kLong, 1, "slots");
    if (slots.size(0) != n) refuse(std::to_string(slots.size(0)) + " slots for " + std::to_string(n) + " tokens");
    int32_t* status = status_of(c, a[6]);
    const Stream stream(c, a[7]);
    check(pf_kv_write(c.index, c.c, k.data, k.token_stride, k.head_stride, v.data, v.token_stride, v.head_stride, *dtype,
                      slots.data_ptr<int64_t>(), uint64_t(n), truth(a[5]), status, stream.raw));
    Py_RETURN_NONE;
  });
}

// read(cache, index, block_table, starts, total, dtype, out, status, stream)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t count) {
  return guarded(count, 9, [&]() -> PyObject* {
    const Cache c = cache(a[0], a[1]);
    const at::Tensor& table = ints(c, a[2], at::kInt, 2, "block_table");
    const at::Tensor& starts = ints(c, a[3], at::kInt, 1, "starts");
    const int64_t seqs = table.size(0), heads = c.c->heads;
    if (starts.size(0) != seqs + 1) {
      refuse(std::to_string(starts.size(0)) + " starts for " + std::to_string(seqs) + " sequences: one more is needed");
    }
    std::optional<at::ScalarType> type;
    if (a[5] != Py_None) {
      if (!THPDtype_Check(a[5])) refuse("dtype must be a torch.dtype");
      type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
    }
    int32_t* status = status_of(c, a[7]);
    const Stream stream(c, a[8]);
    at::Tensor key, value;
    if (a[6] == Py_None) {
      const int64_t total = a[4] == Py_None ? -1 : integer(a[4]);
      if (total < 0) refuse("total, the rows of the result, must be given without out");
      if (!type) type = c.c->dtype == PF_DTYPE_FP16 ? at::kHalf : at::kBFloat16;
      if (!rows_dtype(*type)) refuse(std::string("dtype must be bfloat16, float16 or float32, not ") + at::toString(*type));
      key = made(c, {total, heads, int64_t(c.c->head_dim)}, *type);
      value = made(c, {total, heads, int64_t(c.c->head_dim)}, *type);
    } else {
      if (!PyTuple_Check(a[6]) || PyTuple_GET_SIZE(a[6]) != 2) refuse("out must be (key, value)");
      key = tensor(PyTuple_GET_ITEM(a[6], 0), "key");
      value = tensor(PyTuple_GET_ITEM(a[6], 1), "value");
      if (!rows_dtype(key.scalar_type()) || value.scalar_type() != key.scalar_type()) {
        refuse(std::string("outputs must both be bfloat16, float16 or float32, not ") + at::toString(key.scalar_type()) + " and " +
               at::toString(value.scalar_type()));
      }
      if ((a[4] != Py_None && key.dim() && integer(a[4]) != key.size(0)) || (type && *type != key.scalar_type())) {
        refuse("total or dtype and out differ");
      }
    }
    const int64_t n = key.dim() ? key.size(0) : 0;
    const pf_kv_rows k = rows(c, key, n, heads, "key"), v = rows(c, value, n, heads, "value");
    check(pf_kv_read(c.index, c.c, table.data_ptr<int32_t>(), table.stride(0), uint32_t(table.size(1)), uint32_t(seqs),
                     starts.data_ptr<int32_t>(), k.data, k.token_stride, k.head_stride, v.data, v.token_stride, v.head_stride,
                     *rows_dtype(key.scalar_type()), uint64_t(n), status, stream.raw));
    PyObject* pair = PyTuple_New(2);
    if (!pair) throw PythonError();
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(key)));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(value)));
    return pair;
  });
}

// attend(cache, index, query, block_table, q_start, kv_len, scale, causal, window, max_q, max_kv, out, return_lse,
//        status, stream)
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t count) {
  return guarded(count, 15, [&]() -> PyObject* {
    const Cache c = cache(a[0], a[1]);
    const at::Tensor& query = tensor(a[2], "query");
    const auto dtype = rows_dtype(query.scalar_type());
    if (query.dim() != 3 || !dtype) {
      refuse(std::string("query must be bfloat16 or float16 [n_tokens, q_heads, head_dim], not ") +
             at::toString(query.scalar_type()) + " " + shown(query.sizes()));
    }
    const int64_t n = query.size(0), heads = query.size(1);
    pf_kv_attention x{};
    x.query = rows(c, query, n, heads, "query");
    const at::Tensor& table = ints(c, a[3], at::kInt, 2, "block_table");
    const at::Tensor& q_start = ints(c, a[4], at::kInt, 1, "q_start");
    const at::Tensor& kv_len = ints(c, a[5], at::kInt, 1, "kv_len");
    const int64_t seqs = table.size(0);
    if (q_start.size(0) != seqs + 1 || kv_len.size(0) != seqs) {
      refuse(std::to_string(q_start.size(0)) + " q_start and " + std::to_string(kv_len.size(0)) + " kv_len for " +
             std::to_string(seqs) + " sequences");
    }
    const int64_t window = integer(a[8]), max_q = a[9] == Py_None ? 0 : integer(a[9]), max_kv = a[10] == Py_None ? 0 : integer(a[10]);
    if (window < 0 || max_q < 0 || max_kv < 0) refuse("window, max_q and max_kv cannot be negative");
    int32_t* status = status_of(c, a[13]);
    const Stream stream(c, a[14]);
    at::Tensor out, lse, scratch;
    if (a[11] == Py_None) {
      out = made(c, query.sizes(), query.scalar_type());
    } else {
      out = tensor(a[11], "out");
      if (out.scalar_type() != query.scalar_type()) {
        refuse(std::string("out must be ") + at::toString(query.scalar_type()) + ", not " + at::toString(out.scalar_type()));
      }
    }
    x.out = rows(c, out, n, heads, "out");
    const bool with_lse = truth(a[12]);
    if (with_lse) {
      lse = made(c, {n, heads}, at::kFloat);
      x.lse = reinterpret_cast<uint64_t>(lse.data_ptr());
    }
    x.block_table = reinterpret_cast<uint64_t>(table.data_ptr());
    x.table_stride = table.stride(0);
    x.q_start = reinterpret_cast<uint64_t>(q_start.data_ptr());
    x.kv_len = reinterpret_cast<uint64_t>(kv_len.data_ptr());
    x.status = reinterpret_cast<uint64_t>(status);
    x.n_tokens = uint64_t(n);
    x.n_seqs = uint32_t(seqs);
    x.max_blocks = uint32_t(table.size(1));
    x.q_heads = uint32_t(heads);
    x.dtype = *dtype;
    const auto bound = [](int64_t v) { return uint32_t(std::min<int64_t>(v, INT32_MAX)); };
    x.max_q = bound(max_q);
    x.max_kv = bound(max_kv);
    x.window = bound(window);
    x.scale = a[6] == Py_None ? float(1.0 / std::sqrt(double(c.c->head_dim))) : float(number(a[6]));
    x.causal = truth(a[7]);
    uint64_t need = 0;
    check(pf_kv_attention_workspace(c.index, c.c, &x, &need));
    if (need) {
      scratch = made(c, {int64_t(need)}, at::kByte);
      x.workspace = reinterpret_cast<uint64_t>(scratch.data_ptr());
      x.workspace_bytes = need;
    }
    check(pf_kv_attention_run(c.index, c.c, &x, stream.raw));
    PyObject* result = a[11] == Py_None ? THPVariable_Wrap(std::move(out)) : Py_NewRef(a[11]);
    if (!with_lse) return result;
    PyObject* pair = PyTuple_New(2);
    if (!pair) throw PythonError();
    PyTuple_SET_ITEM(pair, 0, result);
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(lse)));
    return pair;
  });
}

PyMethodDef kMethods[] = {
    {"write", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(write)), METH_FASTCALL, nullptr},
    {"read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(read)), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_kv_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv_torch() { return PyModule_Create(&kModule); }
