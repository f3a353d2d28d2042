// Python binding of the paged-cache operators: takes torch tensors, checks them and calls the C ABI (include/vits_amd.h).
// These calls come once a layer and a token, and their kernels take a few microseconds; the same checks in Python and a ctypes
// call of thirty arguments take six to seven microseconds beside the launch, here one.  vits_amd/ops.py holds the
// interface and its documentation; it passes the current stream and makes the tensors' GPU the current one.
#include <Python.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "../../include/vits_amd.h"

namespace {

using at::Tensor;

// what a caller gets as a ValueError
struct Refused {
  std::string why;
};

// the library's entry points, as its header declares them
decltype(&vits_op_page_plan) plan_fn;
decltype(&vits_op_rotary_store) rotary_fn;
decltype(&vits_op_paged_attention_workspace_bytes) workspace_fn;
decltype(&vits_op_paged_attention) attention_fn;
decltype(&vits_last_error) last_error_fn;
PyObject* vits_error;

std::string describe(const Tensor& t) {
  std::string s = std::string(c10::toString(t.scalar_type())) + " [";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  s += "], strides [";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.stride(i));
  return s + "] on " + t.device().str();
}

const Tensor& tensor(PyObject* o, const char* what, const char* name) {
  if (!THPVariable_Check(o)) throw Refused{std::string(what) + ": " + name + " must be a tensor"};
  return THPVariable_Unpack(o);
}
// a tensor, or null for None
const Tensor* maybe(PyObject* o, const char* what, const char* name) { return o == Py_None ? nullptr : &tensor(o, what, name); }

void flat(const Tensor& t, at::ScalarType type, int64_t n, const char* what, const char* name) {
  if (t.scalar_type() != type || !t.is_contiguous() || (n >= 0 && t.numel() != n))
    throw Refused{std::string(what) + ": " + name + " must be contiguous " + c10::toString(type) + " of " + (n < 0 ? "any number of" : std::to_string(n)) +
                  " elements, got " + describe(t)};
}

int narrow(int64_t x, const char* what) {
  if (x < INT32_MIN || x > INT32_MAX) throw Refused{std::string(what) + ": a size of " + std::to_string(x)};
  return (int)x;
}

int type_of(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kBFloat16: return 2;
    default: throw Refused{std::string(what) + ": values must be fp32, fp16 or bf16, got " + describe(t)};
  }
}

// [rows, heads, dim] with contiguous channels
void rows_of(const Tensor& t, at::ScalarType type, int64_t rows, int64_t heads, int64_t dim, const char* what, const char* name) {
  if (t.scalar_type() != type || t.dim() != 3 || t.size(0) != rows || t.size(1) != heads || t.size(2) != dim || (t.stride(2) != 1 && dim > 1))
    throw Refused{std::string(what) + ": " + name + " must be " + c10::toString(type) + " [" + std::to_string(rows) + ", " + std::to_string(heads) +
                  ", " + std::to_string(dim) + "] with contiguous channels, got " + describe(t)};
}

void caches_of(const Tensor& k, const Tensor& v, const char* what) {
  bool alike = k.dim() == 4 && v.scalar_type() == k.scalar_type() && v.sizes() == k.sizes();
  for (int i = 0; alike && i < 4; ++i) alike = k.size(i) <= 1 || v.stride(i) == k.stride(i);
  if (!alike || k.stride(3) != 1 || k.stride(2) != k.size(3) || (k.stride(1) != k.size(2) * k.size(3) && k.size(1) > 1))
    throw Refused{std::string(what) + ": k_cache and v_cache must be alike, [pages, kv_heads, page_size, dim], and contiguous within a page, got " +
                  describe(k) + " and " + describe(v)};
}

void table_of(const Tensor& t, const char* what) {
  if (t.scalar_type() != at::kInt || t.dim() != 2 || (t.stride(1) != 1 && t.size(1) > 1))
    throw Refused{std::string(what) + ": table must be int32 [requests, width] with contiguous rows, got " + describe(t)};
}

// (the stride of a dimension of one element says nothing)
int64_t page_stride(const Tensor& cache) { return cache.size(0) > 1 ? cache.stride(0) : cache.size(1) * cache.size(2) * cache.size(3); }
int64_t table_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

void no_grad(const char* what, std::initializer_list<const Tensor*> values) {
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode())      // (which torch.no_grad leaves on)
    for (const Tensor* t : values)
      if (t && t->_fw_grad(0).defined())
        throw Refused{std::string(what) + ": carries no tangent along: call it on the primal tensors (torch.autograd.forward_ad.unpack_dual)"};
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : values)
    if (t && t->requires_grad())
      throw Refused{std::string(what) + ": records no gradient: call it under torch.no_grad() (or on detached tensors)"};
}

void on_gpu(const char* what, const Tensor& first, std::initializer_list<const Tensor*> more) {
  if (!first.is_cuda()) throw Refused{std::string(what) + ": tensors must be on a GPU (vits_amd has no CPU path)"};
  for (const Tensor* t : more)
    if (t && t->device() != first.device())
      throw Refused{std::string(what) + ": all tensors must be on one GPU, got " + t->device().str() + " and " + first.device().str()};
}

void* at_(const Tensor* t) { return t ? t->data_ptr() : nullptr; }

long long integer(PyObject* o) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) throw std::exception();
  return x;
}
int integer32(PyObject* o, const char* what) { return narrow(integer(o), what); }
bool truth(PyObject* o) {
  const int x = PyObject_IsTrue(o);
  if (x < 0) throw std::exception();
  return x > 0;
}
double real(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw std::exception();
  return x;
}
void* address(PyObject* o) {
  void* p = PyLong_AsVoidPtr(o);
  if (!p && PyErr_Occurred()) throw std::exception();
  return p;
}

// written: what the call has overwritten.  Autograd learns of that by a tensor's version (inference tensors have none).
PyObject* done(int rc, const char* what, std::initializer_list<const Tensor*> written = {}) {
  if (rc == 0) {
    for (const Tensor* t : written)
      if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
    Py_RETURN_NONE;
  }
  PyErr_Format(vits_error, "%s failed (%d): %s", what, rc, last_error_fn());
  return nullptr;
}

template <typename F>
PyObject* guarded(const char* what, Py_ssize_t got, Py_ssize_t want, F f) {
  try {
    if (got != want) throw Refused{std::string(what) + ": " + std::to_string(want) + " arguments"};
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(PyExc_ValueError, r.why.c_str());
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s: %s", what, e.what());
  }
  return nullptr;
}

// lengths, grow, table, ring, cursor, page_size, rows, out (seven tensors), stream
PyObject* page_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const char* what = "page_plan";
  return guarded(what, n, 9, [&]() -> PyObject* {
    const Tensor &lengths = tensor(a[0], what, "lengths"), &grow = tensor(a[1], what, "grow"), &table = tensor(a[2], what, "table");
    const Tensor &ring = tensor(a[3], what, "ring"), &cursor = tensor(a[4], what, "cursor");
    const int64_t requests = lengths.numel(), rows = integer(a[6]);
    flat(lengths, at::kInt, requests, what, "lengths");
    flat(grow, at::kInt, requests, what, "grow");
    flat(ring, at::kInt, -1, what, "ring");
    flat(cursor, at::kLong, 2, what, "cursor");
    table_of(table, what);
    if (table.size(0) != requests)
      throw Refused{"page_plan: table has " + std::to_string(table.size(0)) + " rows for " + std::to_string(requests) + " requests"};
    static const char* names[7] = {"out.lengths", "out.cursor", "out.start", "out.request", "out.position", "out.slot", "out.status"};
    const int64_t sizes[7] = {requests, 2, requests + 1, rows, rows, rows, 1};
    const Tensor* out[7];
    if (!PyTuple_Check(a[7]) || PyTuple_GET_SIZE(a[7]) != 7) throw Refused{"page_plan: out must hold a PagePlan's seven tensors"};
    for (int i = 0; i < 7; ++i) {
      out[i] = &tensor(PyTuple_GET_ITEM(a[7], i), what, names[i]);
      flat(*out[i], i == 1 || i == 5 ? at::kLong : at::kInt, sizes[i], what, names[i]);
    }
    on_gpu(what, lengths, {&grow, &table, &ring, &cursor, out[0], out[1], out[2], out[3], out[4], out[5], out[6]});
    return done(plan_fn((int*)lengths.data_ptr(), (int*)grow.data_ptr(), narrow(requests, what), (int*)table.data_ptr(), table_stride(table),
                        narrow(table.size(1), what), (int*)ring.data_ptr(), narrow(ring.numel(), what), (int64_t*)cursor.data_ptr(),
                        integer32(a[5], what), (int*)out[0]->data_ptr(), (int64_t*)out[1]->data_ptr(), (int*)out[2]->data_ptr(),
                        (int*)out[3]->data_ptr(), (int*)out[4]->data_ptr(), (int64_t*)out[5]->data_ptr(), narrow(rows, what),
                        (int*)out[6]->data_ptr(), address(a[8])),
                what, {&table, &ring, out[0], out[1], out[2], out[3], out[4], out[5], out[6]});
  });
}

// q, k, v, k_cache, v_cache, position, slot, freq, interleaved, scale, out, err_flag, stream
PyObject* rotary_store(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const char* what = "rotary_store";
  return guarded(what, n, 13, [&]() -> PyObject* {
    const Tensor *q = maybe(a[0], what, "q"), *k = maybe(a[1], what, "k"), *v = maybe(a[2], what, "v");
    const Tensor *kc = maybe(a[3], what, "k_cache"), *vc = maybe(a[4], what, "v_cache"), *slot = maybe(a[6], what, "slot");
    const Tensor *out = maybe(a[10], what, "out"), *flag = maybe(a[11], what, "err_flag");
    const Tensor &position = tensor(a[5], what, "position"), &freq = tensor(a[7], what, "freq");
    const bool interleaved = truth(a[8]);
    const float scale = (float)real(a[9]);
    if (!q && !k) throw Refused{"rotary_store: neither queries nor keys"};
    if (!q && out) throw Refused{"rotary_store: out without q"};
    if (k ? !(v && kc && vc && slot) : v || kc || vc) throw Refused{"rotary_store: keys, values, both caches and slots go together"};
    const Tensor& first = q ? *q : *k;
    const int type = type_of(first, what);
    if (first.dim() != 3) throw Refused{"rotary_store: rows must be [rows, heads, dim], got " + describe(first)};
    const int64_t rows = first.size(0), dim = first.size(2), heads = q ? first.size(1) : 0;
    flat(position, at::kInt, rows, what, "position");
    flat(freq, at::kDouble, -1, what, "freq");
    if (slot) flat(*slot, at::kLong, rows, what, "slot");
    if (flag) flat(*flag, at::kInt, 1, what, "err_flag");
    if (q) {
      rows_of(*q, first.scalar_type(), rows, heads, dim, what, "q");
      rows_of(*out, first.scalar_type(), rows, heads, dim, what, "out");
    }
    if (k) {
      caches_of(*kc, *vc, what);
      rows_of(*k, first.scalar_type(), rows, kc->size(1), dim, what, "k");
      rows_of(*v, first.scalar_type(), rows, kc->size(1), dim, what, "v");
      if (kc->scalar_type() != first.scalar_type() || kc->size(3) != dim)
        throw Refused{"rotary_store: the caches' type and channels are not the rows': " + describe(*kc) + " and " + describe(first)};
    }
    no_grad(what, {q, k, v, kc, vc, &freq, out});
    on_gpu(what, first, {k, v, kc, vc, slot, out, flag, &position, &freq});
    return done(rotary_fn(at_(q), q ? q->stride(0) : 0, q ? q->stride(1) : 0, at_(out), out ? out->stride(0) : 0, out ? out->stride(1) : 0,
                          narrow(heads, what), at_(k), k ? k->stride(0) : 0, k ? k->stride(1) : 0, at_(v), v ? v->stride(0) : 0,
                          v ? v->stride(1) : 0, at_(kc), at_(vc), kc ? page_stride(*kc) : 0, kc ? narrow(kc->size(0), what) : 0,
                          kc ? narrow(kc->size(2), what) : 0, kc ? narrow(kc->size(1), what) : 0, narrow(dim, what), type,
                          (int*)position.data_ptr(), (int64_t*)at_(slot), narrow(rows, what), (double*)freq.data_ptr(),
                          narrow(freq.numel(), what), scale, interleaved, (int*)at_(flag), address(a[12])),
                what, {kc, vc, out, flag});
  });
}

// q, k_cache, v_cache, table, request, position, scale, window, max_keys (0: as many as the table holds), out, lse, err_flag, stream
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const char* what = "paged_attention";
  return guarded(what, n, 13, [&]() -> PyObject* {
    const Tensor &q0 = tensor(a[0], what, "q"), &kc = tensor(a[1], what, "k_cache"), &vc = tensor(a[2], what, "v_cache");
    const Tensor &table = tensor(a[3], what, "table"), &request = tensor(a[4], what, "request"), &position = tensor(a[5], what, "position");
    const Tensor &out = tensor(a[9], what, "out"), *lse = maybe(a[10], what, "lse"), *flag = maybe(a[11], what, "err_flag");
    if (q0.dim() != 3) throw Refused{"paged_attention: q must be [rows, heads, dim], got " + describe(q0)};
    caches_of(kc, vc, what);
    const int type = type_of(kc, what);
    const int64_t rows = q0.size(0), heads = q0.size(1), dim = kc.size(3);
    rows_of(q0, kc.scalar_type(), rows, heads, dim, what, "q");
    rows_of(out, kc.scalar_type(), rows, heads, dim, what, "out");
    flat(request, at::kInt, rows, what, "request");
    flat(position, at::kInt, rows, what, "position");
    table_of(table, what);
    if (lse && (lse->dim() != 2 || lse->size(0) != rows || lse->size(1) != heads || lse->scalar_type() != at::kFloat || !lse->is_contiguous()))
      throw Refused{"paged_attention: lse must be contiguous float32 [rows, heads], got " + describe(*lse)};
    if (flag) flat(*flag, at::kInt, 1, what, "err_flag");
    no_grad(what, {&q0, &kc, &vc, &out, lse});
    on_gpu(what, q0, {&kc, &vc, &table, &request, &position, &out, lse, flag});
    const int64_t size = q0.element_size();
    const bool aligned = ((uintptr_t)q0.data_ptr() | (uintptr_t)(q0.stride(0) * size) | (uintptr_t)(q0.stride(1) * size)) % 16 == 0;
    const Tensor q = aligned ? q0 : q0.clone(at::MemoryFormat::Contiguous);            // the library reads heads on 16-byte addresses
    const int window = integer32(a[7], what);
    int64_t keys = integer(a[8]);
    if (keys <= 0) keys = table.size(1) * kc.size(2);
    if (window > 0 && window < keys) keys = window;
    const int r = narrow(rows, what), h = narrow(heads, what), hk = narrow(kc.size(1), what), d = narrow(dim, what);
    const int64_t bytes = workspace_fn(narrow(table.size(0), what), r, h, hk, d, type, keys);
    if (bytes < 0) return done(-1, what);
    // a workspace of this call's own: calls on different streams, and graphs that run side by side, share none
    Tensor ws;
    if (bytes) ws = at::empty({bytes}, q0.options().dtype(at::kByte));
    return done(attention_fn(q.data_ptr(), q.stride(0), q.stride(1), kc.data_ptr(), vc.data_ptr(), page_stride(kc), narrow(kc.size(0), what),
                             narrow(kc.size(2), what), (int*)table.data_ptr(), table_stride(table), narrow(table.size(1), what),
                             narrow(table.size(0), what), (int*)request.data_ptr(), (int*)position.data_ptr(), r, h, hk, d, type,
                             (float)real(a[6]), window, keys, out.data_ptr(), out.stride(0), out.stride(1), (float*)at_(lse), (int*)at_(flag),
                             bytes ? ws.data_ptr() : nullptr, bytes, address(a[12])),
                what, {&out, lse, flag});
  });
}

// the library's entry points (addresses) and the exception that its errors become
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("bind", n, 6, [&]() -> PyObject* {
    plan_fn = (decltype(plan_fn))address(a[0]);
    rotary_fn = (decltype(rotary_fn))address(a[1]);
    workspace_fn = (decltype(workspace_fn))address(a[2]);
    attention_fn = (decltype(attention_fn))address(a[3]);
    last_error_fn = (decltype(last_error_fn))address(a[4]);
    Py_INCREF(a[5]);
    vits_error = a[5];
    Py_RETURN_NONE;
  });
}

#define METHOD(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(page_plan), METHOD(rotary_store), METHOD(paged_attention), METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_vits_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__vits_ops() { return PyModule_Create(&module); }
