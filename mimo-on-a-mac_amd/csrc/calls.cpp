// The host path of append, read and attend: a decode step makes two of these calls for each layer, of a few microseconds on the
// GPU, and through ctypes and Python's tensor attributes the host takes 8 to 11 for each.  What is here takes the call in its
// ordinary form (tensors of the types and layouts that the kernels read, on the current device, outside of a capture) and
// answers NotImplemented for anything else: mimo_stream/attention.py then checks the arguments one by one, converts what it
// may, and raises what is wrong.  No check is left out here that it makes.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/mimo_moe.h"

namespace {

decltype(&mimo_cache_append_rotary) append_entry = nullptr;
decltype(&mimo_cache_read) read_entry = nullptr;
decltype(&mimo_cache_attend) attend_entry = nullptr;
decltype(&mimo_cache_attend_workspace_size) attend_room = nullptr;

constexpr const char* kCache = "mimo_kv_cache";
struct Cache {
  mimo_kv_cache c;
  int device;
};

PyObject* other() { Py_RETURN_NOTIMPLEMENTED; }

// a plain tensor on the device, or nullptr
const at::Tensor* tensor(PyObject* o, int device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.get_device() == device && t.layout() == at::kStrided && !t.is_neg() ? &t : nullptr;
}
bool int32(const at::Tensor* t) { return t && t->scalar_type() == at::kInt && t->is_contiguous(); }
bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
template <class T> T* at_(const at::Tensor* t) { return static_cast<T*>(t->data_ptr()); }

// rows [N, heads, dim] as the kernels read them: contiguous aligned tokens at any distance, in elements, or -1
int64_t rows(const at::Tensor* t, int64_t heads, int64_t dim) {
  if (!t || t->scalar_type() != at::kBFloat16 || t->dim() != 3 || t->size(2) != dim || (heads >= 0 && t->size(1) != heads)) return -1;
  const int64_t n = t->size(0), h = t->size(1), row = h * dim, s0 = n <= 1 ? row : t->stride(0);
  if (t->stride(2) != 1 || (t->stride(1) != dim && h != 1) || s0 % 8 || s0 < row || !aligned(t->data_ptr())) return -1;
  return s0;
}
at::Tensor bf16(at::IntArrayRef shape, int device) {
  return at::empty(shape, at::TensorOptions().dtype(at::kBFloat16).device(at::Device(at::kCUDA, device)));
}
bool number(PyObject* o, int64_t* x) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  *x = PyLong_AsLongLongAndOverflow(o, &overflow);
  return !overflow;
}
// the status word: None, or int32 [1]; false: something else
bool status_of(PyObject* o, int device, int32_t** status) {
  *status = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = tensor(o, device);
  if (!int32(t) || t->dim() != 1 || t->size(0) != 1) return false;
  *status = at_<int32_t>(t);
  return true;
}
Cache* cache_of(PyObject* o) { return PyCapsule_IsValid(o, kCache) ? static_cast<Cache*>(PyCapsule_GetPointer(o, kCache)) : nullptr; }
// a plan's page size goes with any cache (None) or with those of its own
bool same_pages(PyObject* o, const Cache* c) {
  int64_t page;
  return o == Py_None || (number(o, &page) && page == c->c.page_size);
}

// The entries run without the interpreter's lock, which an exception on its way out would have to have again: no tensor is looked
// at meanwhile, since one without memory of its own (inside of torch.vmap) throws where its address is asked for.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// An exception on its way through C would end the process: an allocation that fails, above all.
template <class F> PyObject* guarded(F f) {
  try {
    return f();
  } catch (const std::exception&) {
    if (PyErr_Occurred()) PyErr_Clear();
    return other();                                        // the long way makes the same allocation, and raises what it raises
  }
}

PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) return PyErr_Format(PyExc_TypeError, "bind takes four addresses");
  void* p[4];
  for (int i = 0; i < 4; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  append_entry = reinterpret_cast<decltype(append_entry)>(p[0]);
  read_entry = reinterpret_cast<decltype(read_entry)>(p[1]);
  attend_entry = reinterpret_cast<decltype(attend_entry)>(p[2]);
  attend_room = reinterpret_cast<decltype(attend_room)>(p[3]);
  Py_RETURN_NONE;
}

// cache(address of a mimo_kv_cache, device index): a copy of the struct; who holds it holds the tensors
PyObject* cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) return PyErr_Format(PyExc_TypeError, "cache takes an address and a device");
  const auto* c = static_cast<const mimo_kv_cache*>(PyLong_AsVoidPtr(a[0]));
  const long device = PyLong_AsLong(a[1]);
  if (PyErr_Occurred()) return nullptr;
  auto* kept = new (std::nothrow) Cache{*c, (int)device};
  if (!kept) return PyErr_NoMemory();
  PyObject* o = PyCapsule_New(kept, kCache, [](PyObject* o) { delete static_cast<Cache*>(PyCapsule_GetPointer(o, kCache)); });
  if (!o) delete kept;
  return o;
}

// append(cache, current device, stream, plan.slots, plan.positions, plan.status, plan.page_size, k, v, q, mimo_rotary address,
// device of its turns): q rotated, None without q, a negative code, or NotImplemented
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 12) return PyErr_Format(PyExc_TypeError, "append takes 12 arguments");
  return guarded([&]() -> PyObject* {
    const Cache* c = cache_of(a[0]);
    int64_t current, stream, rotary, turns;
    if (!c || !number(a[1], &current) || !number(a[2], &stream) || !number(a[10], &rotary) || !number(a[11], &turns)) return other();
    if (current != c->device || !same_pages(a[6], c) || (rotary && turns != c->device)) return other();
    const auto* turn = reinterpret_cast<const mimo_rotary*>(rotary);
    const at::Tensor *slots = tensor(a[3], c->device), *positions = tensor(a[4], c->device), *k = tensor(a[7], c->device), *v = tensor(a[8], c->device);
    const int64_t ks = rows(k, c->c.kv_heads, c->c.k_dim), vs = rows(v, c->c.kv_heads, c->c.v_dim);
    int32_t* status;
    if (ks < 0 || vs < 0 || !int32(slots) || !int32(positions) || !status_of(a[5], c->device, &status)) return other();
    const int64_t N = k->size(0);
    if (N < 1 || N > INT32_MAX || v->size(0) != N || slots->dim() != 1 || slots->size(0) != N || positions->dim() != 1 || positions->size(0) != N) return other();
    const at::Tensor* q = nullptr;
    at::Tensor out;
    int64_t qs = 0, heads = 0;
    if (a[9] != Py_None) {
      q = tensor(a[9], c->device);
      qs = rows(q, -1, c->c.k_dim);
      if (qs < 0 || q->size(0) != N || q->size(1) > 65536) return other();
      heads = q->size(1);
      out = bf16({N, heads, c->c.k_dim}, c->device);
    }
    const uint16_t *at_q = q ? at_<uint16_t>(q) : nullptr, *at_k = at_<uint16_t>(k), *at_v = at_<uint16_t>(v);
    const int32_t *at_positions = at_<int32_t>(positions), *at_slots = at_<int32_t>(slots);
    uint16_t* at_out = q ? at_<uint16_t>(&out) : nullptr;
    const int rc = [&] {
      Unlocked u;
      return append_entry(at_q, qs, (int)heads, at_k, ks, at_v, vs, (int)N, at_positions, at_slots, &c->c, turn, at_out, status,
                          reinterpret_cast<void*>(stream));
    }();
    if (rc) return PyLong_FromLong(rc);
    if (!q) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

// read(cache, current device, stream, slots, status): (k, v), a negative code, or NotImplemented
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5) return PyErr_Format(PyExc_TypeError, "read takes 5 arguments");
  return guarded([&]() -> PyObject* {
    const Cache* c = cache_of(a[0]);
    int64_t current, stream;
    if (!c || !number(a[1], &current) || !number(a[2], &stream) || current != c->device) return other();
    const at::Tensor* slots = tensor(a[3], c->device);
    int32_t* status;
    if (!int32(slots) || slots->dim() != 1 || slots->size(0) < 1 || slots->size(0) > INT32_MAX || !status_of(a[4], c->device, &status)) return other();
    const int64_t N = slots->size(0);
    at::Tensor k = bf16({N, c->c.kv_heads, c->c.k_dim}, c->device), v = bf16({N, c->c.kv_heads, c->c.v_dim}, c->device);
    const int32_t* at_slots = at_<int32_t>(slots);
    uint16_t *at_k = at_<uint16_t>(&k), *at_v = at_<uint16_t>(&v);
    const int rc = [&] {
      Unlocked u;
      return read_entry(&c->c, at_slots, (int)N, at_k, at_v, status, reinterpret_cast<void*>(stream));
    }();
    if (rc) return PyLong_FromLong(rc);
    PyObject *pk = THPVariable_Wrap(std::move(k)), *pv = pk ? THPVariable_Wrap(std::move(v)) : nullptr;
    PyObject* both = pv ? PyTuple_Pack(2, pk, pv) : nullptr;
    Py_XDECREF(pk);
    Py_XDECREF(pv);
    return both;
  });
}

// attend(cache, current device, stream, q, plan.starts, plan.lens, plan.table, plan.max_new, plan.status, plan.page_size, scale,
// window, sink_tokens, sink_logits, out, workspace): out, a negative code, or NotImplemented
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 16) return PyErr_Format(PyExc_TypeError, "attend takes 16 arguments");
  return guarded([&]() -> PyObject* {
    const Cache* c = cache_of(a[0]);
    int64_t current, stream, window, sinks, max_new = -1;
    if (!c || !number(a[1], &current) || !number(a[2], &stream) || current != c->device || !same_pages(a[9], c)) return other();
    if (!number(a[11], &window) || !number(a[12], &sinks) || window < 0 || window > INT32_MAX || sinks < 0 || sinks > INT32_MAX) return other();
    const at::Tensor *q = tensor(a[3], c->device), *starts = tensor(a[4], c->device), *lens = tensor(a[5], c->device), *table = tensor(a[6], c->device);
    const at::Tensor* ws = tensor(a[15], c->device);
    const int64_t qs = rows(q, -1, c->c.k_dim);
    int32_t* status;
    if (qs < 0 || !int32(starts) || !int32(lens) || !int32(table) || !ws || !status_of(a[8], c->device, &status)) return other();
    const int64_t N = q->size(0), heads = q->size(1);
    if (N < 1 || N > (1 << 20) || heads < 1 || heads > INT32_MAX || heads % c->c.kv_heads || table->dim() != 2) return other();
    const int64_t B = table->size(0), width = table->size(1);
    if (B < 1 || B > INT32_MAX || width > INT32_MAX || starts->dim() != 1 || starts->size(0) != B + 1 || lens->dim() != 1 || lens->size(0) != B) return other();
    if (a[7] != Py_None && !number(a[7], &max_new)) return other();
    const int64_t most = a[7] == Py_None ? N : std::max<int64_t>(-1, std::min(N, max_new));
    double scale = 1.0 / std::sqrt((double)c->c.k_dim);
    if (a[10] != Py_None) {
      if (!PyFloat_CheckExact(a[10])) return other();
      scale = PyFloat_AS_DOUBLE(a[10]);
    }
    const float* logits = nullptr;
    if (a[13] != Py_None) {
      const at::Tensor* t = tensor(a[13], c->device);
      if (!t || t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != heads || !t->is_contiguous()) return other();
      logits = at_<float>(t);
    }
    const size_t bytes = (size_t)ws->numel();
    if (ws->scalar_type() != at::kByte || !ws->is_contiguous() || bytes < attend_room((int)N, (int)heads, c->c.kv_heads, c->c.v_dim)) return other();
    at::Tensor made;
    const at::Tensor* out = &made;
    if (a[14] != Py_None) {
      out = tensor(a[14], c->device);
      if (!out || out->scalar_type() != at::kBFloat16 || out->dim() != 3 || out->size(0) != N || out->size(1) != heads || out->size(2) != c->c.v_dim ||
          !out->is_contiguous() || !aligned(out->data_ptr()))
        return other();
    } else {
      made = bf16({N, heads, c->c.v_dim}, c->device);
    }
    const uint16_t* at_q = at_<uint16_t>(q);
    const int32_t *at_starts = at_<int32_t>(starts), *at_lens = at_<int32_t>(lens), *at_table = at_<int32_t>(table);
    uint16_t* at_out = at_<uint16_t>(out);
    void* room = ws->data_ptr();
    const int rc = [&] {
      Unlocked u;
      return attend_entry(at_q, qs, (int)N, (int)heads, &c->c, (int)B, at_starts, at_lens, at_table, (int)width, (int)most, (float)scale,
                          (int)window, (int)sinks, logits, at_out, status, room, bytes, reinterpret_cast<void*>(stream));
    }();
    if (rc) return PyLong_FromLong(rc);
    if (out != &made) {
      Py_INCREF(a[14]);
      return a[14];
    }
    return THPVariable_Wrap(std::move(made));
  });
}

template <class F> PyCFunction fast(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }
PyMethodDef methods[] = {{"bind", fast(bind), METH_FASTCALL, nullptr},     {"cache", fast(cache), METH_FASTCALL, nullptr},
                         {"append", fast(append), METH_FASTCALL, nullptr}, {"read", fast(read), METH_FASTCALL, nullptr},
                         {"attend", fast(attend), METH_FASTCALL, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&module); }
