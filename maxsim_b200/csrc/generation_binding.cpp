// Python entry of the 4-bit cache's and the 4-bit weights' operators (maxsim_b200/generation.py): checks tensors,
// allocates outputs and workspaces through torch, calls the C ABI on torch's current stream.
//
// A decode step calls these a few times per layer with kernels of 3 to 10 us, so the host's part decides: reading
// a tensor's fields here costs a few ns each.  (The same checks in Python over ctypes: 13.9 us a product's call,
// 19.6 us an attention call.)
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "../../include/maxsim_b200.h"

namespace {

struct ValueError {
  std::string message;
};
struct TypeError {
  std::string message;
};
struct PythonError {};  // already set

[[noreturn]] void refuse(const std::string& message) { throw ValueError{message}; }

void check_status(int status) {
  if (status == MSB_OK) return;
  const char* message = msb_last_error();
  PyErr_SetString(status == MSB_ERR_INVALID_ARGUMENT ? PyExc_ValueError
                  : status == MSB_ERR_NOT_SUPPORTED  ? PyExc_NotImplementedError
                                                     : PyExc_RuntimeError,
                  message ? message : "");
  throw PythonError{};
}

std::string text(c10::IntArrayRef sizes) {
  std::string s = "[";
  for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
  return s + "]";
}

const at::Tensor& tensor(PyObject* o, const char* name, c10::Device device) {
  if (!THPVariable_Check(o)) throw TypeError{std::string(name) + " must be a torch tensor"};
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.device() != device) refuse(std::string(name) + " must be on " + device.str() + ", got " + t.device().str());
  return t;
}
void want_dtype(const at::Tensor& t, const char* name, c10::ScalarType type) {
  if (t.scalar_type() != type)
    refuse(std::string(name) + " must have dtype " + c10::toString(type) + ", got " + c10::toString(t.scalar_type()));
}
void want_dim(const at::Tensor& t, const char* name, int64_t dim) {
  if (t.dim() != dim)
    refuse(std::string(name) + " must have " + std::to_string(dim) + " dimensions, got " + std::to_string(t.dim()));
}
// The operators have no backward pass: a result without a history must not pass for one with it.
void no_gradient(const at::Tensor& t, const char* name) {
  if (c10::GradMode::is_enabled() && t.requires_grad())
    refuse(std::string(name) + " requires a gradient, which this operator does not have: call it under torch.no_grad() or on " +
           name + ".detach()");
}
int32_t type_id(c10::ScalarType type, bool f32) {
  if (type == c10::kHalf) return MSB_TYPE_F16;
  if (type == c10::kBFloat16) return MSB_TYPE_BF16;
  if (type == c10::kFloat && f32) return MSB_TYPE_F32;
  refuse(std::string("dtype must be ") + (f32 ? "fp32, fp16 or bf16" : "fp16 or bf16") + ", got " + c10::toString(type));
}
at::Tensor empty(c10::IntArrayRef sizes, c10::ScalarType type, c10::Device device) {
  return at::empty(sizes, c10::TensorOptions().dtype(type).device(device));
}
void* stream_of(c10::Device device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

// Refuses an output (contiguous) that shares memory with what the kernel reads: other blocks may still be reading there.
// `in` is [rows, heads, dim] with any strides but the last; the very same rows in the same places are let through where
// a block writes only what it alone has read (`same_is_fine`).
void no_overlap(const at::Tensor& out, const char* name, const at::Tensor& in, const char* in_name, bool same_is_fine) {
  if (out.numel() == 0 || in.numel() == 0) return;
  const char* const o0 = static_cast<const char*>(out.const_data_ptr());
  const char* const o1 = o0 + out.numel() * out.element_size();
  const char* const i0 = static_cast<const char*>(in.const_data_ptr());
  int64_t last = 0;
  for (int64_t d = 0; d < in.dim(); ++d) last += (in.size(d) - 1) * in.stride(d);
  const int64_t size = in.element_size();
  if (o1 <= i0 || i0 + (last + 1) * size <= o0) return;
  if (same_is_fine && o0 == i0 && in.is_contiguous() && in.numel() == out.numel()) return;
  // The spans meet; the rows may still lie beside the output.
  const int64_t rows = in.size(0), row = in.stride(0) * size, heads = in.dim() == 3 ? in.size(1) : 1;
  const int64_t head = in.dim() == 3 ? in.stride(1) * size : 0, width = in.size(-1) * size;
  for (int64_t r = 0; r < rows; ++r)
    for (int64_t h = 0; h < heads; ++h) {
      const char* const p = i0 + r * row + h * head;
      if (o0 < p + width && p < o1) refuse(std::string(name) + " must not overlap " + in_name);
    }
}

const msb_kv4_cache* cache_of(PyObject* o) {
  void* p = PyLong_AsVoidPtr(o);
  if (PyErr_Occurred()) throw PythonError{};
  return static_cast<const msb_kv4_cache*>(p);
}
c10::Device device_of(int32_t index) { return c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(index)); }
int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PythonError{};
  return v;
}

at::Tensor slots_of(PyObject* o, c10::Device device) {
  const at::Tensor& t = tensor(o, "slots", device);
  want_dtype(t, "slots", c10::kLong);
  want_dim(t, "slots", 1);
  return t.contiguous();
}
at::Tensor vectors_of(PyObject* o, const char* name, const msb_kv4_cache* c, c10::Device device, int64_t tokens) {
  const at::Tensor& t = tensor(o, name, device);
  want_dim(t, name, 3);
  if (t.size(1) != c->kv_heads || t.size(2) != c->head_dim)
    refuse(std::string(name) + " must have shape [tokens, " + std::to_string(c->kv_heads) + ", " +
           std::to_string(c->head_dim) + "], got " + text(t.sizes()));
  if (t.size(0) != tokens) refuse("keys, values and slots must have the same number of tokens");
  return t.stride(2) == 1 ? t : t.contiguous();
}

// append(cache, keys, values, slots)
PyObject* append(PyObject* const* args, Py_ssize_t n) {
  if (n != 4) throw TypeError{"append takes 4 arguments"};
  const msb_kv4_cache* c = cache_of(args[0]);
  const c10::Device device = device_of(c->device);
  const at::Tensor slots = slots_of(args[3], device);
  const at::Tensor keys = vectors_of(args[1], "keys", c, device, slots.size(0));
  const at::Tensor values = vectors_of(args[2], "values", c, device, slots.size(0));
  if (keys.scalar_type() != values.scalar_type()) refuse("keys and values must have the same dtype");
  check_status(msb_kv4_append_device(c, keys.const_data_ptr(), values.const_data_ptr(), type_id(keys.scalar_type(), true),
                                     slots.size(0), keys.stride(0), keys.stride(1), values.stride(0), values.stride(1),
                                     slots.const_data_ptr<int64_t>(), stream_of(device)));
  Py_RETURN_NONE;
}

// read(cache, slots, dtype or None, out or None) -> (keys, values)
PyObject* read(PyObject* const* args, Py_ssize_t n) {
  if (n != 4) throw TypeError{"read takes 4 arguments"};
  const msb_kv4_cache* c = cache_of(args[0]);
  const c10::Device device = device_of(c->device);
  const at::Tensor slots = slots_of(args[1], device);
  const int64_t shape[3] = {slots.size(0), c->kv_heads, c->head_dim};
  c10::ScalarType type = c10::kBFloat16;
  if (args[2] != Py_None) {
    if (!THPDtype_Check(args[2])) throw TypeError{"dtype must be a torch dtype"};
    type = reinterpret_cast<THPDtype*>(args[2])->scalar_type;
  }
  at::Tensor out[2];
  if (args[3] == Py_None) {
    type_id(type, true);
    for (at::Tensor& t : out) t = empty(shape, type, device);
  } else {
    if (!PySequence_Check(args[3]) || PySequence_Size(args[3]) != 2) throw TypeError{"out must be a pair of tensors"};
    static const char* const names[2] = {"out[0]", "out[1]"};
    for (int i = 0; i < 2; ++i) {
      PyObject* item = PySequence_GetItem(args[3], i);
      if (!item) throw PythonError{};
      const bool is_tensor = THPVariable_Check(item);
      if (is_tensor) out[i] = THPVariable_Unpack(item);
      Py_DECREF(item);
      if (!is_tensor) throw TypeError{std::string(names[i]) + " must be a torch tensor"};
      if (out[i].device() != device) refuse(std::string(names[i]) + " must be on " + device.str());
    }
    if (args[2] != Py_None && type != out[0].scalar_type()) refuse("out must have the given dtype");
    type = out[0].scalar_type();
    type_id(type, true);
    for (int i = 0; i < 2; ++i) {
      want_dtype(out[i], names[i], type);
      no_gradient(out[i], names[i]);
      if (!out[i].sizes().equals(shape) || !out[i].is_contiguous())
        refuse(std::string(names[i]) + " must be contiguous with shape " + text(shape));
    }
    no_overlap(out[0], names[0], out[1].view({shape[0], shape[1] * shape[2]}), names[1], false);
  }
  check_status(msb_kv4_read_device(c, slots.const_data_ptr<int64_t>(), shape[0], type_id(type, true),
                                   out[0].mutable_data_ptr(), out[1].mutable_data_ptr(), stream_of(device)));
  PyObject* pair = PyTuple_New(2);
  if (!pair) throw PythonError{};
  for (int i = 0; i < 2; ++i) PyTuple_SET_ITEM(pair, i, THPVariable_Wrap(std::move(out[i])));
  return pair;
}

// attend(cache, query, page_table, lengths, query_offsets, max_query_tokens, scale, causal, window, return_lse, out)
PyObject* attend(PyObject* const* args, Py_ssize_t n) {
  if (n != 11) throw TypeError{"attend takes 11 arguments"};
  const msb_kv4_cache* c = cache_of(args[0]);
  const c10::Device device = device_of(c->device);
  msb_kv4_attend_args a{};
  const at::Tensor& given = tensor(args[1], "query", device);
  want_dim(given, "query", 3);
  no_gradient(given, "query");
  a.type = type_id(given.scalar_type(), false);
  const int64_t rows = given.size(0), heads = given.size(1), dim = given.size(2);
  if (dim != c->head_dim || heads == 0 || heads % c->kv_heads)
    refuse("query must have shape [rows, a multiple of " + std::to_string(c->kv_heads) + ", " +
           std::to_string(c->head_dim) + "], got " + text(given.sizes()));
  const at::Tensor query = given.stride(2) == 1 ? given : given.contiguous();
  const at::Tensor& table = tensor(args[2], "page_table", device);
  want_dtype(table, "page_table", c10::kInt);
  want_dim(table, "page_table", 2);
  const at::Tensor& length = tensor(args[3], "lengths", device);
  want_dtype(length, "lengths", c10::kInt);
  want_dim(length, "lengths", 1);
  const int64_t batch = table.size(0), pages = table.size(1);
  if (length.size(0) != batch) refuse("page_table and lengths must have the same batch");
  if (batch > INT32_MAX || pages > INT32_MAX || heads > INT32_MAX) refuse("sizes must be below 2^31");
  const at::Tensor page_table = pages > 1 && table.stride(1) != 1 ? table.contiguous() : table;
  const at::Tensor lengths = length.contiguous();
  at::Tensor offsets;
  int64_t most = 1;
  if (args[4] == Py_None) {
    if (rows != batch) refuse("without query_offsets, query must have one row per sequence");
    if (args[5] != Py_None && integer(args[5]) != 1) refuse("max_query_tokens needs query_offsets");
  } else {
    const at::Tensor& o = tensor(args[4], "query_offsets", device);
    want_dtype(o, "query_offsets", c10::kInt);
    want_dim(o, "query_offsets", 1);
    if (o.size(0) != batch + 1) refuse("query_offsets must have shape [batch + 1]");
    offsets = o.contiguous();
    most = args[5] == Py_None ? rows : integer(args[5]);
    if (most < 0) refuse("max_query_tokens must not be negative");
    if (most == 0 && rows > 0) refuse("max_query_tokens must be positive where there are rows");
    most = std::min(most, rows);  // a sequence has no more rows than there are
  }
  const int causal = PyObject_IsTrue(args[7]), return_lse = PyObject_IsTrue(args[9]);
  if (causal < 0 || return_lse < 0) throw PythonError{};
  int64_t window = 0;
  if (args[8] != Py_None) {
    window = integer(args[8]);
    if (window < 1 || !causal) refuse("window must be at least 1 and needs causal");
    window = std::min<int64_t>(window, INT32_MAX);
  }
  double scale = 1.0 / std::sqrt(static_cast<double>(dim));
  if (args[6] != Py_None) {
    scale = PyFloat_AsDouble(args[6]);
    if (scale == -1.0 && PyErr_Occurred()) throw PythonError{};
  }
  if (!(static_cast<float>(scale) > 0.0F) || !std::isfinite(static_cast<float>(scale))) refuse("scale must be finite and > 0");
  at::Tensor out;
  const int64_t shape[3] = {rows, heads, dim};
  if (args[10] == Py_None) {
    out = empty(shape, query.scalar_type(), device);
  } else {
    out = tensor(args[10], "out", device);
    want_dtype(out, "out", query.scalar_type());
    if (!out.sizes().equals(shape) || !out.is_contiguous()) refuse("out must be contiguous with shape " + text(shape));
    no_gradient(out, "out");
    no_overlap(out, "out", query, "query", true);
  }
  at::Tensor lse;
  if (return_lse) lse = empty({rows, heads}, c10::kFloat, device);
  a.query = query.const_data_ptr();
  a.query_row_stride = query.stride(0);
  a.query_head_stride = query.stride(1);
  a.rows = rows;
  a.page_table = page_table.const_data_ptr<int32_t>();
  a.page_table_stride = page_table.stride(0);
  a.lengths = lengths.const_data_ptr<int32_t>();
  a.query_offsets = offsets.defined() ? offsets.const_data_ptr<int32_t>() : nullptr;
  a.out = out.mutable_data_ptr();
  a.lse = return_lse ? lse.mutable_data_ptr<float>() : nullptr;
  a.batch = static_cast<int32_t>(batch);
  a.max_pages = static_cast<int32_t>(pages);
  a.max_query_rows = static_cast<int32_t>(std::min<int64_t>(most, INT32_MAX));
  a.heads = static_cast<int32_t>(heads);
  a.causal = causal;
  a.window = static_cast<int32_t>(window);
  a.scale = static_cast<float>(scale);
  int64_t need = 0;
  check_status(msb_kv4_attend_workspace_bytes(c, &a, &need));
  at::Tensor workspace;
  if (need > 0) {
    workspace = empty({need}, c10::kByte, device);
    a.workspace = workspace.mutable_data_ptr();
    a.workspace_bytes = need;
  }
  // Outputs made here are fresh memory: rows that the call does not work on are filled, by the kernel where both are.
  const bool fresh = args[10] == Py_None;
  if (fresh && batch == 0) out.zero_();
  if (return_lse && a.query_offsets && (!fresh || batch == 0)) lse.fill_(-INFINITY);
  check_status((fresh ? msb_kv4_attend_fill_device : msb_kv4_attend_device)(c, &a, stream_of(device)));
  if (!return_lse) return THPVariable_Wrap(std::move(out));
  PyObject* pair = PyTuple_New(2);
  if (!pair) throw PythonError{};
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(out)));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(lse)));
  return pair;
}

// What Int4Linear keeps (mirrored in generation.py).
struct Linear {
  const void* codes;
  const void* scales;
  const void* bias;
  int64_t n;
  int64_t k;
  int32_t group;
  int32_t bias_type;  // MSB_TYPE_*, -1 without a bias
  int32_t device;
};

// linear(handle, x, out or None) -> y
PyObject* linear(PyObject* const* args, Py_ssize_t n) {
  if (n != 3) throw TypeError{"linear takes 3 arguments"};
  const Linear* l = static_cast<const Linear*>(PyLong_AsVoidPtr(args[0]));
  if (PyErr_Occurred()) throw PythonError{};
  const c10::Device device = device_of(l->device);
  const at::Tensor& x = tensor(args[1], "x", device);
  const int32_t type = type_id(x.scalar_type(), false);
  no_gradient(x, "x");
  if (x.dim() < 1 || x.size(-1) != l->k)
    refuse("x must have shape [..., " + std::to_string(l->k) + "], got " + text(x.sizes()));
  if (l->bias_type >= 0 && l->bias_type != type) refuse("bias and x must have the same dtype");
  at::Tensor rows = x.dim() == 2 ? x : x.reshape({-1, l->k});
  if (rows.stride(1) != 1) rows = rows.contiguous();
  // The kernel reads 16 bytes at a time: rows that do not start on 16 bytes are copied.
  if ((reinterpret_cast<uintptr_t>(rows.const_data_ptr()) | static_cast<uint64_t>(rows.stride(0)) * 2) & 15)
    rows = rows.clone(at::MemoryFormat::Contiguous);
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = l->n;
  at::Tensor out;
  if (args[2] == Py_None) {
    out = empty(shape, x.scalar_type(), device);
  } else {
    out = tensor(args[2], "out", device);
    want_dtype(out, "out", x.scalar_type());
    if (!out.sizes().equals(shape) || !out.is_contiguous()) refuse("out must be contiguous with shape " + text(shape));
    no_gradient(out, "out");
    no_overlap(out, "out", rows, "x", false);
  }
  check_status(msb_w4_product_device(l->codes, l->scales, l->n, l->k, l->group, rows.const_data_ptr(), rows.stride(0),
                                     rows.size(0), l->bias, out.mutable_data_ptr(), l->n, type, l->device,
                                     stream_of(device)));
  return THPVariable_Wrap(std::move(out));
}

// Nothing thrown in here leaves as a C++ exception.
template <PyObject* (*kCall)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    return kCall(args, n);
  } catch (const ValueError& e) {
    PyErr_SetString(PyExc_ValueError, e.message.c_str());
  } catch (const TypeError& e) {
    PyErr_SetString(PyExc_TypeError, e.message.c_str());
  } catch (const PythonError&) {
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    PyErr_SetString(type ? type : PyExc_RuntimeError, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

template <PyObject* (*kCall)(PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<kCall>)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<append>("append"), method<read>("read"), method<attend>("attend"),
                         method<linear>("linear"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_generation", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__generation() { return PyModule_Create(&module); }
