// The host's part of a call that is all launch: Python module ringattn_calls, used by api.py.
//
// A forward of a few hundred tokens, or one step of a short ring, is some 5 us of GPU work, and a launch costs the host 4.3 us of
// its own.  The checks of five tensors, their addresses and the stream took Python another 2.2 (6.8 us a call of forward()); here they take
// 0.2 (4.4).  A Call holds one entry point of the C ABI with its plan and the shapes and types it expects.  Called with five tensors and a stream it
// returns the entry point's code, or None, without having done anything, where the arguments are not plainly what it
// expects: the caller then goes the general way, which says what is wrong, or serves what is merely unusual (tensor subclasses).
// Only addresses of this call's tensors are handed on; nothing of a tensor is kept.  A Paged is the same for the paged cache's calls, a Turn for rotary positions, a
// Pages for the bookkeeping of a cache's pages.
#include <Python.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstddef>
#include <new>
#include <vector>

#include "ringattn.h"

namespace {

constexpr int kTensors = 5;
using Fwd = int (*)(void*, const void*, const void*, const void*, void*, void*, void*);
using Step = int (*)(void*, int, int, const void*, const void*, const void*, void*, void*, void*);

struct Spec {
  at::ScalarType type;
  std::vector<int64_t> shape;
};
struct Call {
  PyObject_HEAD
  vectorcallfunc vectorcall;
  void* entry;
  void* plan;
  int rank, step;  // rank < 0: an entry point without them
  std::vector<Spec>* specs;
};

PyObject* call(PyObject* self_, PyObject* const* args, size_t nargsf, PyObject* kwnames) {
  Call* self = reinterpret_cast<Call*>(self_);
  if (PyVectorcall_NARGS(nargsf) != kTensors + 1 || kwnames) {
    PyErr_SetString(PyExc_TypeError, "five tensors and a stream (or None)");
    return nullptr;
  }
  void* p[kTensors];
  hipStream_t stream;
  try {
    for (int i = 0; i < kTensors; ++i) {
      if (!THPVariable_CheckExact(args[i])) Py_RETURN_NONE;
      const at::Tensor& t = THPVariable_Unpack(args[i]);
      const Spec& s = (*self->specs)[i];
      if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || t.scalar_type() != s.type || t.sizes() != s.shape || !t.is_contiguous())
        Py_RETURN_NONE;
      p[i] = t.data_ptr();
    }
    if (args[kTensors] == Py_None) stream = c10::hip::getCurrentHIPStream().stream();
  } catch (...) {  // a tensor without storage, or whose sizes are symbols
    Py_RETURN_NONE;
  }
  if (args[kTensors] != Py_None) {
    PyObject* handle = PyObject_GetAttrString(args[kTensors], "cuda_stream");
    if (!handle) return nullptr;
    stream = static_cast<hipStream_t>(PyLong_AsVoidPtr(handle));
    Py_DECREF(handle);
    if (PyErr_Occurred()) return nullptr;
  }
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (self->rank < 0) rc = reinterpret_cast<Fwd>(self->entry)(self->plan, p[0], p[1], p[2], p[3], p[4], stream);
  else rc = reinterpret_cast<Step>(self->entry)(self->plan, self->rank, self->step, p[0], p[1], p[2], p[3], p[4], stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// Call(address of the entry point, of the plan, rank or -1, step, ((dtype, shape), ... of five tensors))
PyObject* create(PyTypeObject* type, PyObject* args, PyObject* kwargs) {
  unsigned long long entry, plan;
  int rank, step;
  PyObject* specs;
  if (kwargs && PyDict_Size(kwargs) > 0) {
    PyErr_SetString(PyExc_TypeError, "positional arguments only");
    return nullptr;
  }
  if (!PyArg_ParseTuple(args, "KKiiO!", &entry, &plan, &rank, &step, &PyTuple_Type, &specs)) return nullptr;
  if (!entry || PyTuple_GET_SIZE(specs) != kTensors) {
    PyErr_SetString(PyExc_ValueError, "an entry point and five tensors' types and shapes");
    return nullptr;
  }
  Call* self = reinterpret_cast<Call*>(type->tp_alloc(type, 0));
  if (!self) return nullptr;
  self->vectorcall = call;
  self->entry = reinterpret_cast<void*>(static_cast<uintptr_t>(entry));
  self->plan = reinterpret_cast<void*>(static_cast<uintptr_t>(plan));
  self->rank = rank;
  self->step = step;
  try {
    self->specs = new std::vector<Spec>(kTensors);
    for (int i = 0; i < kTensors; ++i) {
      PyObject *dtype, *shape;
      if (!PyArg_ParseTuple(PyTuple_GET_ITEM(specs, i), "OO!", &dtype, &PyTuple_Type, &shape) || !THPDtype_Check(dtype)) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "a torch.dtype and a tuple");
        Py_DECREF(self);
        return nullptr;
      }
      Spec& s = (*self->specs)[i];
      s.type = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
      for (Py_ssize_t j = 0; j < PyTuple_GET_SIZE(shape); ++j) s.shape.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(shape, j)));
      if (PyErr_Occurred()) {
        Py_DECREF(self);
        return nullptr;
      }
    }
  } catch (const std::bad_alloc&) {
    Py_DECREF(self);
    return PyErr_NoMemory();
  }
  return reinterpret_cast<PyObject*>(self);
}

void destroy(PyObject* self) {
  delete reinterpret_cast<Call*>(self)->specs;
  Py_TYPE(self)->tp_free(self);
}

// ---- the paged cache's calls (paged.py): the same for tensors of any strides.  What the caller's Python would check in some 12 us a call
// is checked in one; anything unusual gives None, and paged.py says what is wrong with it or serves it.
struct Paged {
  PyObject_HEAD
  vectorcallfunc vectorcall;
  void* entry;
  void* plan;
  int kind;  // 0 append, 1 forward, 2 weights, 3 evict; 4, 5: 1 and 2 with scores that are shaped; 6: 0 with rotary positions
  int heads, kv_heads, dim, page, max_batch, device;
  long max_tokens;
  at::ScalarType type, out_type;
  float softcap;
};

// A tensor on a device, or nothing.
const at::Tensor* tensor_on(PyObject* o, int device, at::ScalarType type, int64_t dims) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || t.device().index() != device || t.scalar_type() != type || t.dim() != dims) return nullptr;
  return &t;
}
const at::Tensor* tensor_of(PyObject* o, const Paged& p, at::ScalarType type, int64_t dims) { return tensor_on(o, p.device, type, dims); }
// Whole, of these sizes.
bool whole(const at::Tensor& t, std::initializer_list<int64_t> sizes) {
  return t.sizes() == at::IntArrayRef(sizes.begin(), sizes.size()) && t.is_contiguous();
}
// None, or a whole tensor of n entries: whether it is one of the two, and its address.
bool whole_or_none(PyObject* o, int device, at::ScalarType type, int64_t n, void** at) {
  *at = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = tensor_on(o, device, type, 1);
  if (!t || !whole(*t, {n})) return false;
  *at = t->data_ptr();
  return true;
}
// Rows of p.dim that begin at multiples of 16 bytes; the strides of the other dimensions, those of length one as if it were contiguous.
bool rows_of(const at::Tensor& t, int dim, int64_t* strides) {
  const int dims = (int)t.dim();
  const int64_t unit = 16 / (int64_t)t.element_size();
  if (t.size(dims - 1) != dim || t.stride(dims - 1) != 1 || (uintptr_t)t.data_ptr() % 16) return false;
  int64_t step = dim;
  for (int i = dims - 2; i >= 0; --i) {
    const int64_t n = t.size(i), s = n > 1 ? t.stride(i) : step;
    if (n < 1 || s < 0 || s % unit) return false;
    strides[i] = s;
    step = s * n;
  }
  return true;
}
bool rows_of(const at::Tensor& t, const Paged& p, int64_t* strides) { return rows_of(t, p.dim, strides); }
// The stream that a call is to go to; false with a Python error set.
bool stream_of(PyObject* given, hipStream_t* stream) {
  if (given == Py_None) return true;
  PyObject* handle = PyObject_GetAttrString(given, "cuda_stream");
  if (!handle) return false;
  *stream = static_cast<hipStream_t>(PyLong_AsVoidPtr(handle));
  Py_DECREF(handle);
  return !PyErr_Occurred();
}

PyObject* paged_call(PyObject* self_, PyObject* const* args, size_t nargsf, PyObject* kwnames) {
  Paged& p = *reinterpret_cast<Paged*>(self_);
  static constexpr Py_ssize_t kArgs[7] = {9, 9, 8, 12, 12, 11, 14};
  if (PyVectorcall_NARGS(nargsf) != kArgs[p.kind] || kwnames) {
    PyErr_SetString(PyExc_TypeError, "the tensors of the call and a stream (or None)");
    return nullptr;
  }
  PyObject* stream_arg = args[kArgs[p.kind] - 1];
  // where the sequences' tensors are among the arguments
  static constexpr int kCache[7] = {2, 1, 2, 0, 1, 2, 3}, kTable[7] = {4, 3, 3, 3, 3, 3, 5};
  ringattn_paged_cache c{};
  hipStream_t stream = nullptr;
  const bool forward = p.kind == 1 || p.kind == 4, weights = p.kind == 2 || p.kind == 5;
  void* x[6] = {};
  void* masks[3] = {};  // slopes, prefix lengths, first keys
  const ringattn_rotary* rotary = nullptr;
  int64_t a[2] = {}, b[2] = {}, kv[2] = {};
  int tokens = 0, budget = 0, first = 0, last = 0, kept_pages = 0;
  try {
    const at::Tensor* k = tensor_of(args[kCache[p.kind]], p, p.type, 4);
    const at::Tensor* table = tensor_of(args[kTable[p.kind]], p, at::kInt, 2);
    const at::Tensor* lens = tensor_of(args[kTable[p.kind] + 1], p, at::kInt, 1);
    int64_t strides[3], v_strides[3];
    if (!k || !table || !lens || !rows_of(*k, p, strides) || k->size(1) != p.kv_heads || k->size(2) != p.page || k->size(0) > INT32_MAX) Py_RETURN_NONE;
    const int64_t batch = table->size(0), pages = k->size(0);
    if (batch < 1 || batch > p.max_batch || table->size(1) < 1 || table->size(1) > INT32_MAX || !whole(*lens, {batch})) Py_RETURN_NONE;
    if ((table->size(1) > 1 && table->stride(1) != 1) || (batch > 1 && table->stride(0) < table->size(1))) Py_RETURN_NONE;
    c.k = k->data_ptr();
    if (!weights) {
      const at::Tensor* v = tensor_of(args[kCache[p.kind] + 1], p, p.type, 4);
      if (!v || v->sizes() != k->sizes() || !rows_of(*v, p, v_strides)) Py_RETURN_NONE;
      for (int i = 0; i < 3; ++i)
        if (v_strides[i] != strides[i]) Py_RETURN_NONE;
      c.v = v->data_ptr();
    }
    c.page_stride = strides[0];
    c.head_stride = strides[1];
    c.token_stride = strides[2];
    c.pages = (int)pages;
    c.table_pages = (int)table->size(1);
    c.table_stride = batch > 1 ? table->stride(0) : table->size(1);
    c.page_table = table->data_ptr<int>();
    c.kv_lens = lens->data_ptr<int>();
    c.batch = (int)batch;
    if (p.kind != 3) {
      const at::Tensor* starts = tensor_of(args[kTable[p.kind] + 2], p, at::kInt, 1);
      const at::Tensor* rows = tensor_of(args[0], p, p.type, 3);
      if (!starts || !whole(*starts, {batch + 1}) || !rows || rows->size(0) < 1 || rows->size(0) > p.max_tokens) Py_RETURN_NONE;
      if (rows->size(1) != (p.kind == 0 ? p.kv_heads : p.heads) || !rows_of(*rows, p, a)) Py_RETURN_NONE;
      c.q_starts = starts->data_ptr<int>();
      tokens = (int)rows->size(0);
      x[0] = rows->data_ptr();
      if (p.kind == 0) {
        const at::Tensor* v = tensor_of(args[1], p, p.type, 3);
        if (!v || v->sizes() != rows->sizes() || !rows_of(*v, p, b) || a[0] != b[0] || a[1] != b[1]) Py_RETURN_NONE;
        x[1] = v->data_ptr();
        if (args[7] != Py_None) {
          const at::Tensor* scores = tensor_of(args[7], p, at::kFloat, 3);
          if (!scores || !whole(*scores, {pages, p.kv_heads, p.page})) Py_RETURN_NONE;
          x[2] = scores->data_ptr();
        }
      } else if (p.kind == 6) {
        const at::Tensor* k_new = tensor_of(args[1], p, p.type, 3);
        const at::Tensor* v_new = tensor_of(args[2], p, p.type, 3);
        const at::Tensor* out = tensor_of(args[10], p, p.type, 3);
        int64_t of_v[2];
        if (!k_new || !v_new || k_new->size(0) != tokens || k_new->size(1) != p.kv_heads || k_new->sizes() != v_new->sizes() || !rows_of(*k_new, p, kv) ||
            !rows_of(*v_new, p, of_v) || kv[0] != of_v[0] || kv[1] != of_v[1] || !out || out->sizes() != rows->sizes() || !rows_of(*out, p, b))
          Py_RETURN_NONE;
        x[1] = k_new->data_ptr();
        x[2] = v_new->data_ptr();
        x[3] = out->data_ptr();
        if (args[8] != Py_None) {
          const at::Tensor* scores = tensor_of(args[8], p, at::kFloat, 3);
          if (!scores || !whole(*scores, {pages, p.kv_heads, p.page})) Py_RETURN_NONE;
          x[4] = scores->data_ptr();
        }
        if (!whole_or_none(args[9], p.device, at::kInt, tokens, &x[5]) || !PyLong_CheckExact(args[11]) || !tensor_of(args[12], p, at::kLong, 1)) Py_RETURN_NONE;
        rotary = static_cast<const ringattn_rotary*>(PyLong_AsVoidPtr(args[11]));
      } else if (forward) {
        const at::Tensor* out = tensor_of(args[6], p, p.out_type, 3);
        const at::Tensor* lse = tensor_of(args[7], p, at::kFloat, 2);
        if (!out || out->sizes() != rows->sizes() || !rows_of(*out, p, b) || !lse || !whole(*lse, {p.heads, tokens})) Py_RETURN_NONE;
        x[1] = out->data_ptr();
        x[2] = lse->data_ptr();
      } else {
        const at::Tensor* lse = tensor_of(args[1], p, at::kFloat, 2);
        const at::Tensor* scores = tensor_of(args[6], p, at::kFloat, 3);
        if (!lse || !whole(*lse, {p.heads, tokens}) || !scores || !whole(*scores, {pages, p.kv_heads, p.page})) Py_RETURN_NONE;
        x[1] = lse->data_ptr();
        x[2] = scores->data_ptr();
      }
      if (p.kind == 4 || p.kind == 5) {
        PyObject* const* m = args + kArgs[p.kind] - 4;
        if (!whole_or_none(m[0], p.device, at::kFloat, p.heads, &masks[0]) || !whole_or_none(m[1], p.device, at::kInt, batch, &masks[1]) ||
            !whole_or_none(m[2], p.device, at::kInt, tokens, &masks[2]))
          Py_RETURN_NONE;
      }
    } else {
      const at::Tensor* scores = tensor_of(args[2], p, at::kFloat, 3);
      const at::Tensor* kept_table = tensor_of(args[5], p, at::kInt, 2);
      if (!PyLong_CheckExact(args[6]) || !PyLong_CheckExact(args[7]) || !PyLong_CheckExact(args[8])) Py_RETURN_NONE;
      int over[3];
      const long n[3] = {PyLong_AsLongAndOverflow(args[6], over), PyLong_AsLongAndOverflow(args[7], over + 1), PyLong_AsLongAndOverflow(args[8], over + 2)};
      for (int i = 0; i < 3; ++i)
        if (over[i] || n[i] < 0 || n[i] > INT32_MAX) Py_RETURN_NONE;
      const at::Tensor* kept = tensor_of(args[9], p, at::kInt, 3);
      const at::Tensor* kept_lens = tensor_of(args[10], p, at::kInt, 1);
      if (!scores || !whole(*scores, {pages, p.kv_heads, p.page}) || !kept_table || !kept_table->is_contiguous() || kept_table->size(0) != batch ||
          kept_table->size(1) > INT32_MAX || !kept || !whole(*kept, {batch, p.kv_heads, n[0]}) || !kept_lens || !whole(*kept_lens, {batch}))
        Py_RETURN_NONE;
      budget = (int)n[0];
      first = (int)n[1];
      last = (int)n[2];
      kept_pages = (int)kept_table->size(1);
      x[0] = scores->data_ptr();
      x[1] = kept_table->data_ptr();
      x[2] = kept->data_ptr();
      x[3] = kept_lens->data_ptr();
    }
    const auto current = c10::hip::getCurrentHIPStream();
    if (current.device_index() != p.device) Py_RETURN_NONE;
    stream = current.stream();
  } catch (...) {  // a tensor without storage, or whose sizes are symbols
    Py_RETURN_NONE;
  }
  if (!stream_of(stream_arg, &stream)) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  auto* plan = static_cast<ringattn_paged_plan*>(p.plan);
  if (p.kind == 0)
    rc = reinterpret_cast<decltype(&ringattn_paged_append)>(p.entry)(plan, &c, x[0], x[1], tokens, a[0], a[1], (float*)x[2], stream);
  else if (p.kind == 1)
    rc = reinterpret_cast<decltype(&ringattn_paged_fwd)>(p.entry)(plan, &c, x[0], tokens, a[0], a[1], x[1], b[0], b[1], (float*)x[2], stream);
  else if (p.kind == 2)
    rc = reinterpret_cast<decltype(&ringattn_paged_weights)>(p.entry)(plan, &c, x[0], tokens, a[0], a[1], (const float*)x[1], (float*)x[2], stream);
  else if (p.kind == 4 || p.kind == 5) {
    const ringattn_paged_scoring scoring{p.softcap, (const float*)masks[0], (const int*)masks[1], (const int*)masks[2]};
    if (p.kind == 4)
      rc = reinterpret_cast<decltype(&ringattn_paged_fwd_scored)>(p.entry)(plan, &c, &scoring, x[0], tokens, a[0], a[1], x[1], b[0], b[1], (float*)x[2], stream);
    else
      rc = reinterpret_cast<decltype(&ringattn_paged_weights_scored)>(p.entry)(plan, &c, &scoring, x[0], tokens, a[0], a[1], (const float*)x[1], (float*)x[2], stream);
  } else if (p.kind == 6)
    rc = reinterpret_cast<decltype(&ringattn_paged_append_rotary)>(p.entry)(plan, &c, rotary, (const int*)x[5], x[0], a[0], a[1], x[3], b[0], b[1], x[1], x[2],
                                                                          tokens, kv[0], kv[1], (float*)x[4], stream);
  else
    rc = reinterpret_cast<decltype(&ringattn_paged_evict)>(p.entry)(plan, &c, (float*)x[0], (const int*)x[1], kept_pages, kept_pages, budget, first, last,
                                                                   (int*)x[2], (int*)x[3], stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// Paged(address of the entry point, of the plan, kind (0 to 3; 16, 17, 18 for 4, 5, 6), heads, kv_heads, dim, page_size, max_batch, max_tokens, device, dtype, dtype of out[, softcap])
PyObject* paged_create(PyTypeObject* type, PyObject* args, PyObject* kwargs) {
  unsigned long long entry, plan;
  int kind, heads, kv_heads, dim, page, max_batch, max_tokens, device;
  PyObject *dtype, *out_dtype;
  float softcap = 0.f;
  if (kwargs && PyDict_Size(kwargs) > 0) {
    PyErr_SetString(PyExc_TypeError, "positional arguments only");
    return nullptr;
  }
  if (!PyArg_ParseTuple(args, "KKiiiiiiiiOO|f", &entry, &plan, &kind, &heads, &kv_heads, &dim, &page, &max_batch, &max_tokens, &device, &dtype, &out_dtype, &softcap))
    return nullptr;
  const bool known = (kind >= 0 && kind < 4) || (kind >= 16 && kind < 19);
  if (!entry || !known || !THPDtype_Check(dtype) || !THPDtype_Check(out_dtype)) {
    PyErr_SetString(PyExc_ValueError, "an entry point, which of the seven it is, and two torch.dtypes");
    return nullptr;
  }
  Paged* self = reinterpret_cast<Paged*>(type->tp_alloc(type, 0));
  if (!self) return nullptr;
  self->vectorcall = paged_call;
  self->entry = reinterpret_cast<void*>(static_cast<uintptr_t>(entry));
  self->plan = reinterpret_cast<void*>(static_cast<uintptr_t>(plan));
  self->kind = kind < 4 ? kind : kind - 12;
  self->heads = heads;
  self->kv_heads = kv_heads;
  self->dim = dim;
  self->page = page;
  self->max_batch = max_batch;
  self->max_tokens = max_tokens;
  self->device = device;
  self->type = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
  self->out_type = reinterpret_cast<THPDtype*>(out_dtype)->scalar_type;
  self->softcap = softcap;
  return reinterpret_cast<PyObject*>(self);
}

void plain_destroy(PyObject* self) { Py_TYPE(self)->tp_free(self); }

// ---- rotary positions (rotary.py): Turn(q, k or None, positions or None, q_out, k_out or None, inverse, stream or None)
struct Turn {
  PyObject_HEAD
  vectorcallfunc vectorcall;
  void* entry;
  const ringattn_rotary* params[2];  // forth and back: the caller keeps them
  int dim, dtype, device;
  at::ScalarType type;
};

PyObject* turn_call(PyObject* self_, PyObject* const* args, size_t nargsf, PyObject* kwnames) {
  const Turn& p = *reinterpret_cast<Turn*>(self_);
  if (PyVectorcall_NARGS(nargsf) != 7 || kwnames) {
    PyErr_SetString(PyExc_TypeError, "the tensors of the call, whether back, and a stream (or None)");
    return nullptr;
  }
  ringattn_rows rows[2];
  int count = 0;
  int64_t batch = 0, tokens = 0, position_stride = 0;
  void* positions = nullptr;
  hipStream_t stream = nullptr;
  try {
    const int dims = THPVariable_CheckExact(args[0]) ? (int)THPVariable_Unpack(args[0]).dim() : 0;
    if (dims != 3 && dims != 4) Py_RETURN_NONE;
    for (int i = 0; i < 2; ++i) {
      if (i == 1 && args[1] == Py_None) {
        if (args[4] != Py_None) Py_RETURN_NONE;
        break;
      }
      const at::Tensor* in = tensor_on(args[i], p.device, p.type, dims);
      const at::Tensor* out = tensor_on(args[3 + i], p.device, p.type, dims);
      int64_t s[3], o[3];
      if (!in || !out || in->sizes() != out->sizes() || !rows_of(*in, p.dim, s) || !rows_of(*out, p.dim, o)) Py_RETURN_NONE;
      const int64_t b = dims == 4 ? in->size(0) : 1, t = in->size(dims == 4 ? 2 : 0), heads = in->size(1);
      if (b > 65535 || t > 1 << 30 || heads > 65535 || (i == 1 && (b != batch || t != tokens))) Py_RETURN_NONE;
      batch = b;
      tokens = t;
      if (dims == 4) rows[i] = ringattn_rows{in->data_ptr(), out->data_ptr(), (int)heads, s[0], s[1], s[2], o[0], o[1], o[2]};
      else rows[i] = ringattn_rows{in->data_ptr(), out->data_ptr(), (int)heads, 0, s[1], s[0], 0, o[1], o[0]};
      ++count;
    }
    if (args[2] != Py_None) {
      if (dims == 4 && THPVariable_CheckExact(args[2]) && THPVariable_Unpack(args[2]).dim() == 2) {
        const at::Tensor* x = tensor_on(args[2], p.device, at::kInt, 2);
        if (!x || !whole(*x, {batch, tokens})) Py_RETURN_NONE;
        positions = x->data_ptr();
        position_stride = tokens;
      } else if (!whole_or_none(args[2], p.device, at::kInt, tokens, &positions)) Py_RETURN_NONE;
    }
    const auto current = c10::hip::getCurrentHIPStream();
    if (current.device_index() != p.device) Py_RETURN_NONE;
    stream = current.stream();
  } catch (...) {
    Py_RETURN_NONE;
  }
  const int back = PyObject_IsTrue(args[5]);
  if (back < 0 || !stream_of(args[6], &stream)) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = reinterpret_cast<decltype(&ringattn_rotary_apply)>(p.entry)(p.params[back], p.dim, p.dtype, rows, count, (int)batch, (int)tokens, (const int*)positions,
                                                                 position_stride, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// Turn(address of the entry point, of the parameters forth, back, dim, RINGATTN_DTYPE_*, device, dtype)
PyObject* turn_create(PyTypeObject* type, PyObject* args, PyObject*) {
  unsigned long long entry, forth, back;
  int dim, code, device;
  PyObject* dtype;
  if (!PyArg_ParseTuple(args, "KKKiiiO", &entry, &forth, &back, &dim, &code, &device, &dtype)) return nullptr;
  if (!entry || !forth || !back || !THPDtype_Check(dtype)) {
    PyErr_SetString(PyExc_ValueError, "an entry point, its parameters, and a torch.dtype");
    return nullptr;
  }
  Turn* self = reinterpret_cast<Turn*>(type->tp_alloc(type, 0));
  if (!self) return nullptr;
  self->vectorcall = turn_call;
  self->entry = reinterpret_cast<void*>(static_cast<uintptr_t>(entry));
  self->params[0] = reinterpret_cast<const ringattn_rotary*>(static_cast<uintptr_t>(forth));
  self->params[1] = reinterpret_cast<const ringattn_rotary*>(static_cast<uintptr_t>(back));
  self->dim = dim;
  self->dtype = code;
  self->device = device;
  self->type = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
  return reinterpret_cast<PyObject*>(self);
}

// ---- pages (paged.PagePool): Pages(k, v, scores or None, parents or None, add or None, short, stream or None), or with kind 1
// Pages(k, v, scores or None, moved or None, None, used, stream or None); calls that ask for pairs go the general way
struct Pages {
  PyObject_HEAD
  vectorcallfunc vectorcall;
  void* entry;
  const ringattn_pages* pages;  // the caller keeps it
  int kind, device;
};

PyObject* pages_call(PyObject* self_, PyObject* const* args, size_t nargsf, PyObject* kwnames) {
  const Pages& p = *reinterpret_cast<Pages*>(self_);
  if (PyVectorcall_NARGS(nargsf) != 7 || kwnames) {
    PyErr_SetString(PyExc_TypeError, "the tensors of the call and a stream (or None)");
    return nullptr;
  }
  ringattn_paged_pool pool{};
  void* x[3] = {};
  hipStream_t stream = nullptr;
  try {
    if (!THPVariable_CheckExact(args[0])) Py_RETURN_NONE;
    const at::ScalarType type = THPVariable_Unpack(args[0]).scalar_type();
    if (type != at::kHalf && type != at::kBFloat16) Py_RETURN_NONE;
    const at::Tensor* k = tensor_on(args[0], p.device, type, 4);
    const at::Tensor* v = tensor_on(args[1], p.device, type, 4);
    int64_t s[3], of_v[3];
    if (!k || !v || k->sizes() != v->sizes() || k->size(0) != p.pages->pages || k->size(2) != p.pages->page_size || k->size(1) > 65535 || k->size(3) > 128 ||
        !rows_of(*k, (int)k->size(3), s) || !rows_of(*v, (int)k->size(3), of_v) || s[0] != of_v[0] || s[1] != of_v[1] || s[2] != of_v[2])
      Py_RETURN_NONE;
    pool = ringattn_paged_pool{k->data_ptr(), v->data_ptr(), nullptr, s[0], s[1], s[2], (int)k->size(1), (int)k->size(3)};
    if (args[2] != Py_None) {
      const at::Tensor* scores = tensor_on(args[2], p.device, at::kFloat, 3);
      if (!scores || !whole(*scores, {k->size(0), k->size(1), k->size(2)})) Py_RETURN_NONE;
      pool.scores = scores->data_ptr<float>();
    }
    const int64_t rows = p.pages->rows, n[2][3] = {{rows, rows, rows}, {p.pages->pages, 0, 1}};
    for (int i = 0; i < 3; ++i)
      if (!whole_or_none(args[3 + i], p.device, at::kInt, n[p.kind][i], &x[i])) Py_RETURN_NONE;
    if (!x[2]) Py_RETURN_NONE;
    const auto current = c10::hip::getCurrentHIPStream();
    if (current.device_index() != p.device) Py_RETURN_NONE;
    stream = current.stream();
  } catch (...) {
    Py_RETURN_NONE;
  }
  if (!stream_of(args[6], &stream)) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (p.kind == 0)
    rc = reinterpret_cast<decltype(&ringattn_pages_update)>(p.entry)(p.pages, &pool, (const int*)x[0], (const int*)x[1], (int*)x[2], nullptr, stream);
  else
    rc = reinterpret_cast<decltype(&ringattn_pages_compact)>(p.entry)(p.pages, &pool, (int*)x[2], (int*)x[0], nullptr, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// Pages(address of the entry point, of the ringattn_pages, 0: update or 1: compact, device)
PyObject* pages_create(PyTypeObject* type, PyObject* args, PyObject*) {
  unsigned long long entry, pages;
  int kind, device;
  if (!PyArg_ParseTuple(args, "KKii", &entry, &pages, &kind, &device)) return nullptr;
  if (!entry || !pages || kind < 0 || kind > 1) {
    PyErr_SetString(PyExc_ValueError, "an entry point, which of the two it is, and its pages");
    return nullptr;
  }
  Pages* self = reinterpret_cast<Pages*>(type->tp_alloc(type, 0));
  if (!self) return nullptr;
  self->vectorcall = pages_call;
  self->entry = reinterpret_cast<void*>(static_cast<uintptr_t>(entry));
  self->pages = reinterpret_cast<const ringattn_pages*>(static_cast<uintptr_t>(pages));
  self->kind = kind;
  self->device = device;
  return reinterpret_cast<PyObject*>(self);
}

PyTypeObject call_type = {PyVarObject_HEAD_INIT(nullptr, 0)};
PyTypeObject paged_type = {PyVarObject_HEAD_INIT(nullptr, 0)};
PyTypeObject turn_type = {PyVarObject_HEAD_INIT(nullptr, 0)};
PyTypeObject pages_type = {PyVarObject_HEAD_INIT(nullptr, 0)};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ringattn_calls", "checks and launch of a call", -1};

}  // namespace

PyMODINIT_FUNC PyInit_ringattn_calls() {
  struct Made {
    PyTypeObject& type;
    const char *name, *in_module;
    Py_ssize_t size, vectorcall;
    destructor destroy;
    newfunc create;
  };
  const Made made[] = {{call_type, "ringattn_calls.Call", "Call", sizeof(Call), offsetof(Call, vectorcall), destroy, create},
                       {paged_type, "ringattn_calls.Paged", "Paged", sizeof(Paged), offsetof(Paged, vectorcall), plain_destroy, paged_create},
                       {turn_type, "ringattn_calls.Turn", "Turn", sizeof(Turn), offsetof(Turn, vectorcall), plain_destroy, turn_create},
                       {pages_type, "ringattn_calls.Pages", "Pages", sizeof(Pages), offsetof(Pages, vectorcall), plain_destroy, pages_create}};
  for (const Made& m : made) {
    m.type.tp_name = m.name;
    m.type.tp_basicsize = m.size;
    m.type.tp_dealloc = m.destroy;
    m.type.tp_vectorcall_offset = m.vectorcall;
    m.type.tp_call = PyVectorcall_Call;
    m.type.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL;
    m.type.tp_new = m.create;
    if (PyType_Ready(&m.type) < 0) return nullptr;
  }
  PyObject* module_ = PyModule_Create(&module);
  if (!module_) return nullptr;
  for (const Made& m : made) {
    Py_INCREF(&m.type);
    if (PyModule_AddObject(module_, m.in_module, reinterpret_cast<PyObject*>(&m.type)) < 0) {
      Py_DECREF(&m.type);
      Py_DECREF(module_);
      return nullptr;
    }
  }
  return module_;
}
