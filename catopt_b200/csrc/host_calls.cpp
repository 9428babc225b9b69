// The checks and the launch of a paged-cache call in one step, for calls whose time is the host's: with some fourteen
// tensors, attribute reads in Python take about 13 us and the foreign call's conversions 3 us (an append of one token to
// 64 requests: 20.2 -> 6.1 us a call; the kernel 3.9).  A function here takes over a call that is in order as it stands;
// for any other (a refusal to word, rows to copy, a device to prepare) it returns NotImplemented, and the wrapper in
// ops.py, which states the rules, goes through it.  Returns what the wrapper returns, or the status code of an entry
// point that declined.  Nothing is remembered between calls.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <climits>

#include "../../include/catopt_b200.h"

namespace {

using at::Tensor;

struct NotTaken {};

const Tensor* tensor(PyObject* o, int dev) {
  if (!THPVariable_CheckExact(o)) throw NotTaken{};
  const Tensor* t = &THPVariable_Unpack(o);
  if (!t->is_cuda() || t->get_device() != dev || t->layout() != at::kStrided || (t->requires_grad() && c10::GradMode::is_enabled()) ||
      t->_fw_grad(0).defined())
    throw NotTaken{};
  return t;
}
void need(bool ok) {
  if (!ok) throw NotTaken{};
}
long long integer(PyObject* o) {
  need(PyLong_CheckExact(o));
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw NotTaken{};
  }
  return x;
}
int bounded(PyObject* o, long long most) {
  const long long x = integer(o);
  need(x >= 0 && x <= most);
  return int(x);
}
bool truth(PyObject* o) {
  need(o == Py_True || o == Py_False);
  return o == Py_True;
}
float real(PyObject* o) {
  need(PyFloat_CheckExact(o));
  return float(PyFloat_AS_DOUBLE(o));
}
template <class T>
T* dense(PyObject* o, int dev, at::ScalarType type, at::IntArrayRef shape) {
  const Tensor* t = tensor(o, dev);
  need(t->scalar_type() == type && t->sizes() == shape && t->is_contiguous());
  return static_cast<T*>(t->data_ptr());
}
template <class T>
T* dense_or_null(PyObject* o, int dev, at::ScalarType type, at::IntArrayRef shape) {
  return o == Py_None ? nullptr : dense<T>(o, dev, type, shape);
}

struct Pools {
  const Tensor* k;
  const Tensor* v;
  long long n, hkv, ps, d, ks, vs;
  int dtype;
};
Pools pools(PyObject* ko, PyObject* vo, int dev) {
  Pools p;
  p.k = tensor(ko, dev);
  p.v = tensor(vo, dev);
  need(p.k->dim() == 4 && p.k->sizes() == p.v->sizes() && p.k->scalar_type() == p.v->scalar_type() && p.k->numel() > 0);
  need(p.k->scalar_type() == at::kFloat || p.k->scalar_type() == at::kBFloat16);
  p.dtype = p.k->scalar_type() == at::kFloat ? CB2_F32 : CB2_BF16;
  p.n = p.k->size(0), p.hkv = p.k->size(1), p.ps = p.k->size(2), p.d = p.k->size(3);
  need(p.n <= INT_MAX && p.hkv <= INT_MAX && p.ps <= 1024 && p.d <= 128);
  for (const Tensor* t : {p.k, p.v}) {
    const long long page = p.hkv * p.ps * p.d, step = p.n > 1 ? t->stride(0) : page;      // of one page, the stride says nothing
    need(t->stride(3) == 1 && t->stride(2) == p.d && t->stride(1) == p.ps * p.d && step >= page);
    (t == p.k ? p.ks : p.vs) = step;
  }
  if (p.k == p.v) p.vs = p.ks;
  return p;
}

struct Rows {
  const Tensor* t;
  const void* at;
  long long token, head;
};
// [n, heads, d] read in place
Rows rows(PyObject* o, int dev, const Pools& p) {
  Rows r{tensor(o, dev), nullptr, 0, 0};
  need(r.t->dim() == 3 && r.t->scalar_type() == p.k->scalar_type() && r.t->size(2) == p.d && r.t->size(0) <= INT_MAX && r.t->size(1) <= INT_MAX);
  const long long unit = 16 / r.t->element_size();
  r.at = r.t->data_ptr();
  r.token = r.t->stride(0), r.head = r.t->stride(1);
  need(r.t->numel() > 0 && r.t->stride(2) == 1 && r.token % unit == 0 && r.head % unit == 0 && r.token && r.head && reinterpret_cast<uintptr_t>(r.at) % 16 == 0);
  return r;
}

int device() { return int(c10::cuda::current_device()); }

// the device's status word; its first call, which makes it, is the wrapper's
int* status(PyObject* words, int dev) {
  PyObject* key = PyLong_FromLong(dev);
  PyObject* w = key ? PyDict_GetItem(words, key) : nullptr;
  Py_XDECREF(key);
  need(w && THPVariable_Check(w));
  return static_cast<int*>(THPVariable_Unpack(w).data_ptr());
}
void* stream(int dev) { return c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(dev)).stream(); }

// Others may run Python while memory is found and kernels are launched.
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

PyObject* declined() { Py_RETURN_NOTIMPLEMENTED; }

// No exception leaves a function of the module; what torch throws (out of memory) the wrapper meets again and raises.
template <class F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (...) {
    return declined();
  }
}

// (words, q, k, v, k_pages, v_pages, table, lens, cu, q_weight, k_weight, eps, cos, sin, positions, interleaved, weights, out)
PyObject* paged_append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    need(n_args == 18);
    const int dev = device();
    const Pools p = pools(a[4], a[5], dev);
    const at::ScalarType dt = p.k->scalar_type();
    const Tensor* bt = tensor(a[6], dev);
    need(bt->dim() == 2 && bt->numel() > 0 && bt->size(0) < INT_MAX && bt->size(1) <= INT_MAX);
    const long long R = bt->size(0), max_pages = bt->size(1);
    const int* table = dense<int>(a[6], dev, at::kInt, {R, max_pages});
    const int* lens = dense<int>(a[7], dev, at::kInt, {R});
    const int* cu = dense<int>(a[8], dev, at::kInt, {R + 1});
    const Rows k = rows(a[2], dev, p), v = rows(a[3], dev, p);
    const long long n = k.t->size(0);
    need(k.t->size(1) == p.hkv && v.t->sizes() == k.t->sizes());
    void* qw = dense_or_null<void>(a[9], dev, dt, {p.d});
    void* kw = dense_or_null<void>(a[10], dev, dt, {p.d});
    float* w = dense_or_null<float>(a[16], dev, at::kFloat, {p.n, p.hkv, p.ps});
    const float *cos = nullptr, *sin = nullptr;
    const int* pos = nullptr;
    long long table_rows = 0, half = 0;
    if (a[12] != Py_None || a[13] != Py_None) {
      const Tensor* c = tensor(a[12], dev);
      need(c->dim() == 2 && c->numel() > 0 && 2 * c->size(1) <= p.d && c->size(0) <= INT_MAX);
      table_rows = c->size(0), half = c->size(1);
      cos = dense<float>(a[12], dev, at::kFloat, {table_rows, half});
      sin = dense<float>(a[13], dev, at::kFloat, {table_rows, half});
      pos = dense<int>(a[14], dev, at::kInt, {n});
    }
    Rows q{nullptr, nullptr, 0, 0};
    void* to = nullptr;
    if (a[1] != Py_None) {
      q = rows(a[1], dev, p);
      need(q.t->size(0) == n);
      to = dense_or_null<void>(a[17], dev, dt, q.t->sizes());
    }
    const float eps = real(a[11]);
    const bool interleaved = truth(a[15]);
    int* word = status(a[0], dev);
    Tensor res;
    int rc;
    {
      const NoGil no_gil;
      if (q.t && !to) res = at::empty(q.t->sizes(), at::TensorOptions(q.t->device()).dtype(dt)), to = res.data_ptr();
      rc = cb2_paged_append(q.at, q.token, q.head, k.at, k.token, k.head, v.at, v.token, v.head, to, p.k->data_ptr(), p.v->data_ptr(), p.ks,
                            p.vs, w, table, lens, cu, pos, qw, kw, eps, cos, sin, int(table_rows), int(2 * half), interleaved, int(n), int(R),
                            q.t ? int(q.t->size(1)) : 0, int(p.hkv), int(p.d), int(p.ps), int(p.n), int(max_pages), p.dtype, word, stream(dev));
    }
    if (rc != CB2_OK) return PyLong_FromLong(rc);
    if (res.defined()) return THPVariable_Wrap(res);
    PyObject* given = q.t ? a[17] : Py_None;
    Py_INCREF(given);
    return given;
  });
}

// (words, q, k_pages, v_pages, table, lens, cu, max_q, max_k, scale, causal, weights, out)
PyObject* om_paged_fwd(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    need(n_args == 13);
    const int dev = device();
    const Pools p = pools(a[2], a[3], dev);
    const at::ScalarType dt = p.k->scalar_type();
    const Tensor* bt = tensor(a[4], dev);
    need(bt->dim() == 2 && bt->numel() > 0 && bt->size(0) < INT_MAX && bt->size(1) <= INT_MAX);
    const long long R = bt->size(0), max_pages = bt->size(1);
    const int* table = dense<int>(a[4], dev, at::kInt, {R, max_pages});
    const int* lens = dense<int>(a[5], dev, at::kInt, {R});
    const int* cu = dense<int>(a[6], dev, at::kInt, {R + 1});
    const Rows q = rows(a[1], dev, p);
    const long long n = q.t->size(0), hq = q.t->size(1), most = std::min(max_pages * p.ps, 1ll << 30);
    need(hq % p.hkv == 0);
    float* w = dense_or_null<float>(a[11], dev, at::kFloat, {p.n, p.hkv, p.ps});
    const int max_q = bounded(a[7], INT_MAX);
    need(a[8] != Py_None || max_pages * p.ps <= most);
    const int max_k = a[8] == Py_None ? int(max_pages * p.ps) : bounded(a[8], most);
    const float scale = a[9] == Py_None ? float(std::pow(double(p.d), -0.5)) : real(a[9]);
    const bool causal = truth(a[10]);
    int* word = status(a[0], dev);
    void* o = dense_or_null<void>(a[12], dev, dt, q.t->sizes());
    Tensor res;
    int rc;
    {
      const NoGil no_gil;
      if (!o) res = at::empty(q.t->sizes(), at::TensorOptions(q.t->device()).dtype(dt)), o = res.data_ptr();
      const size_t bytes = cb2_om_paged_scratch_bytes(int(n), int(R), int(hq), int(p.hkv), int(p.d), max_q, max_k, w != nullptr, p.dtype);
      // a buffer of its own for every call: two captured graphs, or two streams, never share one
      const Tensor scratch = at::empty({std::max((long long)(bytes), 16ll)}, at::TensorOptions(q.t->device()).dtype(at::kByte));
      rc = cb2_om_paged_fwd(q.at, q.token, q.head, p.k->data_ptr(), p.v->data_ptr(), p.ks, p.vs, o, w, table, lens, cu, int(n), int(R), int(hq),
                            int(p.hkv), int(p.d), int(p.ps), int(p.n), int(max_pages), max_q, max_k, scale, causal, p.dtype, scratch.data_ptr(),
                            bytes, word, stream(dev));
    }
    if (rc != CB2_OK) return PyLong_FromLong(rc);
    if (res.defined()) return THPVariable_Wrap(res);
    Py_INCREF(a[12]);
    return a[12];
  });
}

// (words, k_pages, v_pages, weights, table, lens, new_table, budget, keep_first, keep_last, max_k)
PyObject* paged_evict(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    need(n_args == 11);
    const int dev = device();
    const Pools p = pools(a[1], a[2], dev);
    float* w = dense<float>(a[3], dev, at::kFloat, {p.n, p.hkv, p.ps});
    const Tensor *bt = tensor(a[4], dev), *nt = tensor(a[6], dev);
    need(bt->dim() == 2 && bt->numel() > 0 && nt->dim() == 2 && nt->numel() > 0 && bt->size(0) < INT_MAX && bt->size(1) <= INT_MAX && nt->size(1) <= INT_MAX);
    const long long R = bt->size(0), max_pages = bt->size(1), new_pages = nt->size(1), most = std::min(max_pages * p.ps, 1ll << 30);
    const int* table = dense<int>(a[4], dev, at::kInt, {R, max_pages});
    const int* lens = dense<int>(a[5], dev, at::kInt, {R});
    const int* to = dense<int>(a[6], dev, at::kInt, {R, new_pages});
    const int budget = bounded(a[7], 1 << 30), first = bounded(a[8], budget), last = bounded(a[9], budget);
    need(budget >= 1 && new_pages * p.ps >= budget && (a[10] != Py_None || max_pages * p.ps <= most));
    const int max_k = a[10] == Py_None ? int(max_pages * p.ps) : bounded(a[10], most);
    int* word = status(a[0], dev);
    Tensor kept, new_lens;
    int rc;
    {
      const NoGil no_gil;
      const at::TensorOptions opt = at::TensorOptions(p.k->device()).dtype(at::kInt);
      kept = at::empty({R, p.hkv, budget}, opt);
      new_lens = at::empty({R}, opt);
      rc = cb2_paged_evict(p.k->data_ptr(), p.v->data_ptr(), p.ks, p.vs, w, table, lens, to, kept.data_ptr<int>(), new_lens.data_ptr<int>(), int(R),
                           int(p.hkv), int(p.d), int(p.ps), int(p.n), int(max_pages), int(new_pages), max_k, budget, first, last, p.dtype, word,
                           stream(dev));
    }
    if (rc != CB2_OK) return PyLong_FromLong(rc);
    PyObject *x = THPVariable_Wrap(kept), *y = THPVariable_Wrap(new_lens);
    PyObject* both = x && y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return both;
  });
}

PyMethodDef kMethods[] = {
    {"paged_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_append)), METH_FASTCALL, nullptr},
    {"om_paged_fwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(om_paged_fwd)), METH_FASTCALL, nullptr},
    {"paged_evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(paged_evict)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&kModule); }
