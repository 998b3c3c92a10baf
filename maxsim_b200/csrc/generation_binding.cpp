// Python entry of the operators of a reader model (maxsim_b200/generation.py): checks tensors,
// allocates outputs and workspaces through torch, calls the C ABI on torch's current stream.
//
// A decode step calls these a few times per layer with kernels of 3 to 10 us, so the host's part decides: reading
// a tensor's fields here costs a few ns each.  (The same checks in Python over ctypes: 13.9 us a product's call,
// 19.6 us an attention call.)
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <optional>
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
// (at::empty comes here through two dispatches, 0.15 us a tensor.  Dispatch modes do not see these tensors, nor are they filled
// where torch fills uninitialised memory: every element of an output is written.)
at::Tensor empty(c10::IntArrayRef sizes, c10::ScalarType type, c10::Device device) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
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

PyObject* pair_of(at::Tensor first, at::Tensor second) {
  PyObject* pair = PyTuple_New(2);
  if (!pair) throw PythonError{};
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(first)));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(second)));
  return pair;
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

at::Tensor slots_of(PyObject* o, c10::Device device, const char* name = "slots") {
  const at::Tensor& t = tensor(o, name, device);
  want_dtype(t, name, c10::kLong);
  want_dim(t, name, 1);
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
  return pair_of(std::move(out[0]), std::move(out[1]));
}

// move(cache, source, target)
PyObject* move(PyObject* const* args, Py_ssize_t n) {
  if (n != 3) throw TypeError{"move takes 3 arguments"};
  const msb_kv4_cache* c = cache_of(args[0]);
  const c10::Device device = device_of(c->device);
  const at::Tensor source = slots_of(args[1], device, "source"), target = slots_of(args[2], device, "target");
  if (source.size(0) != target.size(0)) refuse("source and target must have the same number of tokens");
  int64_t need = 0;
  check_status(msb_kv4_move_workspace_bytes(c, source.size(0), &need));
  at::Tensor workspace;
  if (need > 0) workspace = empty({need}, c10::kByte, device);
  check_status(msb_kv4_move_device(c, source.const_data_ptr<int64_t>(), target.const_data_ptr<int64_t>(), source.size(0),
                                   need > 0 ? workspace.mutable_data_ptr() : nullptr, need, stream_of(device)));
  Py_RETURN_NONE;
}

// attend(cache, query, page_table, lengths, query_offsets, max_query_tokens, scale, causal, window, sinks, ancestors,
//        return_lse, out)
PyObject* attend(PyObject* const* args, Py_ssize_t n) {
  if (n != 13) throw TypeError{"attend takes 13 arguments"};
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
  const int causal = PyObject_IsTrue(args[7]), return_lse = PyObject_IsTrue(args[11]);
  if (causal < 0 || return_lse < 0) throw PythonError{};
  int64_t window = 0;
  if (args[8] != Py_None) {
    window = integer(args[8]);
    if (window < 1 || !causal) refuse("window must be at least 1 and needs causal");
    window = std::min<int64_t>(window, INT32_MAX);
  }
  msb_kv4_attend_mask mask{};
  const int64_t sinks = integer(args[9]);
  if (sinks < 0) refuse("sinks must not be negative");
  if (sinks > 0 && window == 0) refuse("sinks need a window");
  mask.sinks = static_cast<int32_t>(std::min<int64_t>(sinks, INT32_MAX));
  at::Tensor ancestors;
  if (args[10] != Py_None) {
    const at::Tensor& t = tensor(args[10], "ancestors", device);
    want_dtype(t, "ancestors", c10::kLong);
    want_dim(t, "ancestors", 2);
    if (t.size(0) != rows || t.size(1) < 1)
      refuse("ancestors must have shape [" + std::to_string(rows) + ", words], got " + text(t.sizes()));
    if (t.size(1) > (1 << 24)) refuse("ancestors must have at most 2^24 words");
    if (!causal || args[4] == Py_None) refuse("ancestors need causal and query_offsets");
    ancestors = t.size(1) > 1 && t.stride(1) != 1 ? t.contiguous() : t;
    mask.ancestors = ancestors.const_data_ptr<int64_t>();
    mask.ancestors_stride = ancestors.stride(0);
    mask.ancestor_words = static_cast<int32_t>(ancestors.size(1));
  }
  const bool masked = mask.sinks > 0 || ancestors.defined();
  double scale = 1.0 / std::sqrt(static_cast<double>(dim));
  if (args[6] != Py_None) {
    scale = PyFloat_AsDouble(args[6]);
    if (scale == -1.0 && PyErr_Occurred()) throw PythonError{};
  }
  if (!(static_cast<float>(scale) > 0.0F) || !std::isfinite(static_cast<float>(scale))) refuse("scale must be finite and > 0");
  at::Tensor out;
  const int64_t shape[3] = {rows, heads, dim};
  if (args[12] == Py_None) {
    out = empty(shape, query.scalar_type(), device);
  } else {
    out = tensor(args[12], "out", device);
    want_dtype(out, "out", query.scalar_type());
    if (!out.sizes().equals(shape) || !out.is_contiguous()) refuse("out must be contiguous with shape " + text(shape));
    no_gradient(out, "out");
    no_overlap(out, "out", query, "query", true);
    if (ancestors.defined()) no_overlap(out, "out", ancestors, "ancestors", false);
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
  check_status(masked ? msb_kv4_attend_masked_workspace_bytes(c, &a, &mask, &need) : msb_kv4_attend_workspace_bytes(c, &a, &need));
  at::Tensor workspace;
  if (need > 0) {
    workspace = empty({need}, c10::kByte, device);
    a.workspace = workspace.mutable_data_ptr();
    a.workspace_bytes = need;
  }
  // Outputs made here are fresh memory: rows that the call does not work on are filled, by the kernel where both are.
  const bool fresh = args[12] == Py_None;
  if (fresh && batch == 0) out.zero_();
  if (return_lse && a.query_offsets && (!fresh || batch == 0)) lse.fill_(-INFINITY);
  check_status(masked ? msb_kv4_attend_masked_device(c, &a, &mask, fresh, stream_of(device))
                      : (fresh ? msb_kv4_attend_fill_device : msb_kv4_attend_device)(c, &a, stream_of(device)));
  if (!return_lse) return THPVariable_Wrap(std::move(out));
  return pair_of(std::move(out), std::move(lse));
}

// draft_ancestors(parents, query_offsets, max_query_tokens or None) -> (ancestors, depths)
PyObject* draft_ancestors(PyObject* const* args, Py_ssize_t n) {
  if (n != 3) throw TypeError{"draft_ancestors takes 3 arguments"};
  if (!THPVariable_Check(args[0])) throw TypeError{"parents must be a torch tensor"};
  const at::Tensor& given = THPVariable_Unpack(args[0]);
  const c10::Device device = given.device();
  if (device.type() != c10::kCUDA) refuse("parents must be on a CUDA device, got " + device.str());
  want_dtype(given, "parents", c10::kInt);
  want_dim(given, "parents", 1);
  const at::Tensor& starts = tensor(args[1], "query_offsets", device);
  want_dtype(starts, "query_offsets", c10::kInt);
  want_dim(starts, "query_offsets", 1);
  if (starts.size(0) < 1) refuse("query_offsets must have shape [batch + 1]");
  const int64_t rows = given.size(0), batch = starts.size(0) - 1;
  if (batch > INT32_MAX) refuse("sizes must be below 2^31");
  int64_t most = args[2] == Py_None ? rows : integer(args[2]);
  if (most < 0) refuse("max_query_tokens must not be negative");
  most = std::min(most, rows);
  if (most > 1024) refuse("a sequence's tree has at most 1024 rows: give max_query_tokens where sequences share the rows");
  const int64_t words = std::max<int64_t>(1, (most + 63) / 64);
  const at::Tensor parents = given.contiguous(), offsets = starts.contiguous();
  at::Tensor ancestors = empty({rows, words}, c10::kLong, device), depths = empty({rows}, c10::kInt, device);
  check_status(msb_draft_ancestors_device(parents.const_data_ptr<int32_t>(), rows, offsets.const_data_ptr<int32_t>(),
                                          static_cast<int32_t>(batch), static_cast<int32_t>(most),
                                          static_cast<int32_t>(words), ancestors.mutable_data_ptr<int64_t>(),
                                          depths.mutable_data_ptr<int32_t>(), device.index(), stream_of(device)));
  return pair_of(std::move(ancestors), std::move(depths));
}

const msb_page_table* pages_of(PyObject* o) {
  void* p = PyLong_AsVoidPtr(o);
  if (PyErr_Occurred()) throw PythonError{};
  return static_cast<const msb_page_table*>(p);
}
// int32 [sequences], apart from what the call writes (its own lengths themselves are fine: each is read first).
at::Tensor per_sequence(PyObject* o, const char* name, const msb_page_table* t, c10::Device device) {
  const at::Tensor& x = tensor(o, name, device);
  want_dtype(x, name, c10::kInt);
  if (x.dim() != 1 || x.size(0) != t->sequences)
    refuse(std::string(name) + " must have shape [" + std::to_string(t->sequences) + "], got " + text(x.sizes()));
  const at::Tensor r = x.contiguous();
  const char* const p = static_cast<const char*>(r.const_data_ptr());
  const auto meets = [&](const int32_t* q, int64_t count) {
    const char* const c = reinterpret_cast<const char*>(q);
    return p < c + 4 * count && c < p + 4 * static_cast<int64_t>(t->sequences);
  };
  if (meets(t->page_table, static_cast<int64_t>(t->sequences) * t->max_pages) || meets(t->free_pages, t->num_pages) ||
      meets(t->free_count, 1) || (r.const_data_ptr() != t->lengths && meets(t->lengths, t->sequences)))
    refuse(std::string(name) + " must not overlap the page table's arrays");
  return r;
}
at::Tensor pages_workspace(const msb_page_table* t, int64_t rows, c10::Device device, int64_t& need) {
  check_status(msb_pages_workspace_bytes(t, rows, &need));
  at::Tensor workspace;
  if (need > 0) workspace = empty({need}, c10::kByte, device);
  return workspace;
}

// extend(table, tokens, rows) -> (query_offsets, slots, positions)
PyObject* extend(PyObject* const* args, Py_ssize_t n) {
  if (n != 3) throw TypeError{"extend takes 3 arguments"};
  const msb_page_table* t = pages_of(args[0]);
  const c10::Device device = device_of(t->device);
  const at::Tensor tokens = per_sequence(args[1], "tokens", t, device);
  const int64_t rows = integer(args[2]);
  if (rows < 0 || rows > INT32_MAX) refuse("rows must be from 0 to 2^31 - 1");
  at::Tensor offsets = empty({static_cast<int64_t>(t->sequences) + 1}, c10::kInt, device);
  at::Tensor slots = empty({rows}, c10::kLong, device), positions = empty({rows}, c10::kInt, device);
  int64_t need = 0;
  at::Tensor workspace = pages_workspace(t, rows, device, need);
  check_status(msb_pages_extend_device(t, tokens.const_data_ptr<int32_t>(), rows, offsets.mutable_data_ptr<int32_t>(),
                                       slots.mutable_data_ptr<int64_t>(), positions.mutable_data_ptr<int32_t>(),
                                       need > 0 ? workspace.mutable_data_ptr() : nullptr, need, stream_of(device)));
  PyObject* triple = PyTuple_New(3);
  if (!triple) throw PythonError{};
  PyTuple_SET_ITEM(triple, 0, THPVariable_Wrap(std::move(offsets)));
  PyTuple_SET_ITEM(triple, 1, THPVariable_Wrap(std::move(slots)));
  PyTuple_SET_ITEM(triple, 2, THPVariable_Wrap(std::move(positions)));
  return triple;
}

// truncate(table, lengths)
PyObject* truncate(PyObject* const* args, Py_ssize_t n) {
  if (n != 2) throw TypeError{"truncate takes 2 arguments"};
  const msb_page_table* t = pages_of(args[0]);
  const c10::Device device = device_of(t->device);
  const at::Tensor lengths = per_sequence(args[1], "lengths", t, device);
  int64_t need = 0;
  at::Tensor workspace = pages_workspace(t, 0, device, need);
  check_status(msb_pages_truncate_device(t, lengths.const_data_ptr<int32_t>(),
                                         need > 0 ? workspace.mutable_data_ptr() : nullptr, need, stream_of(device)));
  Py_RETURN_NONE;
}

// What Rotary keeps (mirrored in generation.py).
struct RotaryHandle {
  msb_rotary table;
  int32_t axes;
};
// Vectors of a rotary call: [tokens, heads, dim] with the last dimension contiguous, in bytes.
struct Vectors {
  const char* at;
  int64_t tokens, heads, token, head, width;
};
Vectors vectors(const at::Tensor& t) {
  const int64_t size = t.element_size();
  return {static_cast<const char*>(t.const_data_ptr()), t.size(0), t.size(1), t.size(0) > 1 ? t.stride(0) * size : 0,
          t.size(1) > 1 ? t.stride(1) * size : 0, t.size(2) * size};
}
int64_t span(const Vectors& v) { return (v.tokens - 1) * v.token + (v.heads - 1) * v.head + v.width; }
// Whether [a, a + na) and [b, b + nb), repeated every `period` bytes, stay apart.
bool apart_every(int64_t period, int64_t from_a_to_b, int64_t na, int64_t nb) {
  if (period <= 0) return false;
  const int64_t d = ((from_a_to_b % period) + period) % period;
  return d >= na && d + nb <= period;
}
// Whether two sets of vectors are seen to lie apart: by their spans, or as parts of rows (or of heads) of one array.
bool apart(const Vectors& a, const Vectors& b) {
  if (a.at + span(a) <= b.at || b.at + span(b) <= a.at) return true;
  const int64_t d = b.at - a.at;
  const auto inner = [](const Vectors& v, bool tokens) {
    return tokens ? (v.heads - 1) * v.head + v.width : (v.tokens - 1) * v.token + v.width;
  };
  if (a.token == b.token && apart_every(a.token, d, inner(a, true), inner(b, true))) return true;
  if (a.head == b.head && apart_every(a.head, d, inner(a, false), inner(b, false))) return true;
  // Both strides alike, one a multiple of the other: parts of the same vectors.
  const int64_t lo = std::min(a.token, a.head), hi = std::max(a.token, a.head);
  return a.token == b.token && a.head == b.head && lo > 0 && hi % lo == 0 && apart_every(lo, d, a.width, b.width);
}
bool written_once(const Vectors& v) {
  const bool tokens_in = v.token < v.head;
  const int64_t in = tokens_in ? v.token : v.head, n = tokens_in ? v.tokens : v.heads;
  const int64_t out = tokens_in ? v.head : v.token, m = tokens_in ? v.heads : v.tokens;
  return (n <= 1 || in >= v.width) && (m <= 1 || out >= (n - 1) * in + v.width);
}
bool same(const Vectors& a, const Vectors& b) { return a.at == b.at && a.token == b.token && a.head == b.head; }

// rotate(handle, query, keys or None, positions, inverse, out or None) -> (query, keys or None)
PyObject* rotate(PyObject* const* args, Py_ssize_t n) {
  if (n != 6) throw TypeError{"rotate takes 6 arguments"};
  const RotaryHandle* handle = static_cast<const RotaryHandle*>(PyLong_AsVoidPtr(args[0]));
  if (PyErr_Occurred()) throw PythonError{};
  const msb_rotary& table = handle->table;
  const c10::Device device = device_of(table.device);
  static const char* const names[2] = {"query", "keys"};
  static const char* const out_names[2] = {"out[0]", "out[1]"};
  msb_rotate_args a{};
  at::Tensor x[2], y[2];
  int count = 0;
  for (int w = 0; w < 2; ++w) {
    if (w == 1 && args[2] == Py_None) continue;
    const at::Tensor& t = tensor(args[1 + w], names[w], device);
    want_dim(t, names[w], 3);
    no_gradient(t, names[w]);
    if (t.size(2) != table.head_dim)
      refuse(std::string(names[w]) + " must have shape [tokens, heads, " + std::to_string(table.head_dim) + "], got " + text(t.sizes()));
    if (w == 1 && t.scalar_type() != x[0].scalar_type()) refuse("query and keys must have the same dtype");
    if (w == 1 && t.size(0) != x[0].size(0)) refuse("query and keys must have the same number of tokens");
    if (t.size(1) > 65535) refuse("heads must be at most 65535");
    x[w] = t;
    ++count;
  }
  const int64_t tokens = x[0].size(0);
  a.type = type_id(x[0].scalar_type(), true);
  const at::Tensor& given = tensor(args[3], "positions", device);
  if (given.scalar_type() != c10::kLong && given.scalar_type() != c10::kInt)
    refuse(std::string("positions must have dtype Int or Long, got ") + c10::toString(given.scalar_type()));
  const bool flat = given.dim() == 1 && handle->axes == 1;
  if (!flat && (given.dim() != 2 || given.size(0) != handle->axes))
    refuse("positions must have shape [" + std::to_string(handle->axes) + ", tokens], got " + text(given.sizes()));
  if (given.size(flat ? 0 : 1) != tokens) refuse("positions and query must have the same number of tokens");
  const int inverse = PyObject_IsTrue(args[4]);
  if (inverse < 0) throw PythonError{};
  if (args[5] == Py_None) {
    for (int w = 0; w < count; ++w) y[w] = empty(x[w].sizes(), x[w].scalar_type(), device);
  } else {
    if (!PySequence_Check(args[5]) || PySequence_Size(args[5]) != 2) throw TypeError{"out must be a pair of tensors"};
    for (int w = 0; w < 2; ++w) {
      PyObject* item = PySequence_GetItem(args[5], w);
      if (!item) throw PythonError{};
      const bool none = item == Py_None, is_tensor = THPVariable_Check(item);
      if (is_tensor) y[w] = THPVariable_Unpack(item);
      Py_DECREF(item);
      if (w == 1 && count == 1) {
        if (!none) refuse("out[1] must be None where keys are");
        continue;
      }
      if (!is_tensor) throw TypeError{std::string(out_names[w]) + " must be a torch tensor"};
      if (y[w].device() != device) refuse(std::string(out_names[w]) + " must be on " + device.str());
      want_dtype(y[w], out_names[w], x[w].scalar_type());
      no_gradient(y[w], out_names[w]);
      if (!y[w].sizes().equals(x[w].sizes()) || (y[w].stride(2) != 1 && y[w].size(2) > 1))
        refuse(std::string(out_names[w]) + " must have shape " + text(x[w].sizes()) + " with contiguous dimensions");
    }
    for (int w = 0; w < count && tokens > 0; ++w) {
      if (y[w].numel() == 0) continue;
      const Vectors out = vectors(y[w]);
      if (!written_once(out)) refuse(std::string(out_names[w]) + " must not overlap itself");
      for (int i = 0; i < count; ++i) {
        if (x[i].numel() == 0) continue;
        const bool in_place = i == w && x[i].stride(2) == 1 && same(out, vectors(x[i]));
        // (An input with other strides in its vectors is copied first, but its memory is written nonetheless.)
        if (!in_place && x[i].stride(2) == 1 && !apart(out, vectors(x[i])))
          refuse(std::string(out_names[w]) + " must be " + names[w] + " itself or lie apart from " + names[i]);
        if (i > w && y[i].numel() > 0 && !apart(out, vectors(y[i]))) refuse("out[0] and out[1] must lie apart");
      }
      int64_t last = 0;
      for (int64_t d = 0; d < given.dim(); ++d) last += (given.size(d) - 1) * given.stride(d);
      const char* const p = static_cast<const char*>(given.const_data_ptr());
      if (p < out.at + span(out) && out.at < p + (last + 1) * static_cast<int64_t>(given.element_size()))
        refuse(std::string(out_names[w]) + " must lie apart from positions");
    }
  }
  for (int w = 0; w < count; ++w) {
    if (x[w].stride(2) != 1 && x[w].size(2) > 1) x[w] = x[w].contiguous();
    a.x[w] = x[w].const_data_ptr();
    a.y[w] = y[w].mutable_data_ptr();
    // Strides of a single token or head are never used, and say nothing of alignment.
    a.x_token_stride[w] = tokens > 1 ? x[w].stride(0) : 0;
    a.y_token_stride[w] = tokens > 1 ? y[w].stride(0) : 0;
    a.x_head_stride[w] = x[w].size(1) > 1 ? x[w].stride(1) : 0;
    a.y_head_stride[w] = x[w].size(1) > 1 ? y[w].stride(1) : 0;
    a.heads[w] = static_cast<int32_t>(x[w].size(1));
  }
  a.positions = given.const_data_ptr();
  a.position_axis_stride = flat ? 0 : given.stride(0);
  a.position_token_stride = given.stride(flat ? 0 : 1);
  a.wide_positions = given.scalar_type() == c10::kLong;
  a.tokens = tokens;
  a.inverse = inverse;
  check_status(msb_rotate_device(&table, &a, stream_of(device)));
  PyObject* pair = PyTuple_New(2);
  if (!pair) throw PythonError{};
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(y[0])));
  if (count == 1) Py_INCREF(Py_None);
  PyTuple_SET_ITEM(pair, 1, count == 1 ? Py_None : THPVariable_Wrap(std::move(y[1])));
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
                         method<linear>("linear"), method<move>("move"), method<draft_ancestors>("draft_ancestors"),
                         method<extend>("extend"), method<truncate>("truncate"), method<rotate>("rotate"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_generation", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__generation() { return PyModule_Create(&module); }
