// The host's part of a call that is all launch: Python module ringattn_calls, used by api.py.
//
// A forward of a few hundred tokens, or one step of a short ring, is some 5 us of GPU work, and a launch costs the host 4.3 us of
// its own.  The checks of five tensors, their addresses and the stream took Python another 2.2 (6.8 us a call of forward()); here they take
// 0.2 (4.4).  A Call holds one entry point of the C ABI with its plan and the shapes and types it expects.  Called with five tensors and a stream it
// returns the entry point's code, or None, without having done anything, where the arguments are not plainly what it
// expects: the caller then goes the general way, which says what is wrong, or serves what is merely unusual (tensor subclasses).
// Only addresses of this call's tensors are handed on; nothing of a tensor is kept.  A Paged is the same for the paged cache's calls.
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
  int kind;  // 0 append, 1 forward, 2 weights, 3 evict
  int heads, kv_heads, dim, page, max_batch, device;
  long max_tokens;
  at::ScalarType type, out_type;
};

// A tensor on the plan's device, or nothing.
const at::Tensor* tensor_of(PyObject* o, const Paged& p, at::ScalarType type, int64_t dims) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || t.device().index() != p.device || t.scalar_type() != type || t.dim() != dims) return nullptr;
  return &t;
}
// Whole, of these sizes.
bool whole(const at::Tensor& t, std::initializer_list<int64_t> sizes) {
  return t.sizes() == at::IntArrayRef(sizes.begin(), sizes.size()) && t.is_contiguous();
}
// Rows of p.dim that begin at multiples of 16 bytes; the strides of the other dimensions, those of length one as if it were contiguous.
bool rows_of(const at::Tensor& t, const Paged& p, int64_t* strides) {
  const int dims = (int)t.dim();
  const int64_t unit = 16 / (int64_t)t.element_size();
  if (t.size(dims - 1) != p.dim || t.stride(dims - 1) != 1 || (uintptr_t)t.data_ptr() % 16) return false;
  int64_t step = p.dim;
  for (int i = dims - 2; i >= 0; --i) {
    const int64_t n = t.size(i), s = n > 1 ? t.stride(i) : step;
    if (n < 1 || s < 0 || s % unit) return false;
    strides[i] = s;
    step = s * n;
  }
  return true;
}

PyObject* paged_call(PyObject* self_, PyObject* const* args, size_t nargsf, PyObject* kwnames) {
  Paged& p = *reinterpret_cast<Paged*>(self_);
  static constexpr Py_ssize_t kArgs[4] = {9, 9, 8, 12};
  if (PyVectorcall_NARGS(nargsf) != kArgs[p.kind] || kwnames) {
    PyErr_SetString(PyExc_TypeError, "the tensors of the call and a stream (or None)");
    return nullptr;
  }
  PyObject* stream_arg = args[kArgs[p.kind] - 1];
  // where the sequences' tensors are among the arguments
  static constexpr int kCache[4] = {2, 1, 2, 0}, kTable[4] = {4, 3, 3, 3};
  ringattn_paged_cache c{};
  hipStream_t stream = nullptr;
  void* x[6] = {};
  int64_t a[2] = {}, b[2] = {};
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
    if (p.kind != 2) {
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
      } else if (p.kind == 1) {
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
  if (stream_arg != Py_None) {
    PyObject* handle = PyObject_GetAttrString(stream_arg, "cuda_stream");
    if (!handle) return nullptr;
    stream = static_cast<hipStream_t>(PyLong_AsVoidPtr(handle));
    Py_DECREF(handle);
    if (PyErr_Occurred()) return nullptr;
  }
  int rc;
  Py_BEGIN_ALLOW_THREADS
  auto* plan = static_cast<ringattn_paged_plan*>(p.plan);
  if (p.kind == 0)
    rc = reinterpret_cast<decltype(&ringattn_paged_append)>(p.entry)(plan, &c, x[0], x[1], tokens, a[0], a[1], (float*)x[2], stream);
  else if (p.kind == 1)
    rc = reinterpret_cast<decltype(&ringattn_paged_fwd)>(p.entry)(plan, &c, x[0], tokens, a[0], a[1], x[1], b[0], b[1], (float*)x[2], stream);
  else if (p.kind == 2)
    rc = reinterpret_cast<decltype(&ringattn_paged_weights)>(p.entry)(plan, &c, x[0], tokens, a[0], a[1], (const float*)x[1], (float*)x[2], stream);
  else
    rc = reinterpret_cast<decltype(&ringattn_paged_evict)>(p.entry)(plan, &c, (float*)x[0], (const int*)x[1], kept_pages, kept_pages, budget, first, last,
                                                                   (int*)x[2], (int*)x[3], stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// Paged(address of the entry point, of the plan, kind, heads, kv_heads, dim, page_size, max_batch, max_tokens, device, dtype, dtype of out)
PyObject* paged_create(PyTypeObject* type, PyObject* args, PyObject* kwargs) {
  unsigned long long entry, plan;
  int kind, heads, kv_heads, dim, page, max_batch, max_tokens, device;
  PyObject *dtype, *out_dtype;
  if (kwargs && PyDict_Size(kwargs) > 0) {
    PyErr_SetString(PyExc_TypeError, "positional arguments only");
    return nullptr;
  }
  if (!PyArg_ParseTuple(args, "KKiiiiiiiiOO", &entry, &plan, &kind, &heads, &kv_heads, &dim, &page, &max_batch, &max_tokens, &device, &dtype, &out_dtype))
    return nullptr;
  if (!entry || kind < 0 || kind > 3 || !THPDtype_Check(dtype) || !THPDtype_Check(out_dtype)) {
    PyErr_SetString(PyExc_ValueError, "an entry point, which of the four it is, and two torch.dtypes");
    return nullptr;
  }
  Paged* self = reinterpret_cast<Paged*>(type->tp_alloc(type, 0));
  if (!self) return nullptr;
  self->vectorcall = paged_call;
  self->entry = reinterpret_cast<void*>(static_cast<uintptr_t>(entry));
  self->plan = reinterpret_cast<void*>(static_cast<uintptr_t>(plan));
  self->kind = kind;
  self->heads = heads;
  self->kv_heads = kv_heads;
  self->dim = dim;
  self->page = page;
  self->max_batch = max_batch;
  self->max_tokens = max_tokens;
  self->device = device;
  self->type = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
  self->out_type = reinterpret_cast<THPDtype*>(out_dtype)->scalar_type;
  return reinterpret_cast<PyObject*>(self);
}

void paged_destroy(PyObject* self) { Py_TYPE(self)->tp_free(self); }

PyTypeObject call_type = {PyVarObject_HEAD_INIT(nullptr, 0)};
PyTypeObject paged_type = {PyVarObject_HEAD_INIT(nullptr, 0)};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ringattn_calls", "checks and launch of a call", -1};

}  // namespace

PyMODINIT_FUNC PyInit_ringattn_calls() {
  call_type.tp_name = "ringattn_calls.Call";
  call_type.tp_basicsize = sizeof(Call);
  call_type.tp_dealloc = destroy;
  call_type.tp_vectorcall_offset = offsetof(Call, vectorcall);
  call_type.tp_call = PyVectorcall_Call;
  call_type.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL;
  call_type.tp_new = create;
  paged_type.tp_name = "ringattn_calls.Paged";
  paged_type.tp_basicsize = sizeof(Paged);
  paged_type.tp_dealloc = paged_destroy;
  paged_type.tp_vectorcall_offset = offsetof(Paged, vectorcall);
  paged_type.tp_call = PyVectorcall_Call;
  paged_type.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL;
  paged_type.tp_new = paged_create;
  if (PyType_Ready(&call_type) < 0 || PyType_Ready(&paged_type) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module);
  if (!m) return nullptr;
  Py_INCREF(&paged_type);
  if (PyModule_AddObject(m, "Paged", reinterpret_cast<PyObject*>(&paged_type)) < 0) {
    Py_DECREF(&paged_type);
    Py_DECREF(m);
    return nullptr;
  }
  Py_INCREF(&call_type);
  if (PyModule_AddObject(m, "Call", reinterpret_cast<PyObject*>(&call_type)) < 0) {
    Py_DECREF(&call_type);
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
