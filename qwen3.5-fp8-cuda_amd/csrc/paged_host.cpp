// The host side of PagedKVCache's calls (paged.py): checks the torch tensors of a call and
// launches it.  A decode step calls these a layer, and eager Python spends longer on the
// attributes of eleven tensors than the kernel takes (a write of one token: 9.4 us a call with
// the checks in Python, the GPU idle for half of it; 5.4 with these, of which the kernel 4.9).
//
// Each function takes the addresses of the C entry point and of its descriptors, which the
// Python object keeps, and the call's tensors; it returns the entry point's status, or None
// where a tensor is not what the call takes: paged.py then finds out which, for the message.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <exception>

#include <torch/csrc/autograd/python_variable.h>

#include "../../include/qwen35_fp8_hip.h"

namespace {

// A call's tensors: each check notes a misfit and hands back what the entry point takes.
struct Args {
  PyObject* const* v;
  int dev = -1;
  bool good = true;

  const at::Tensor* tensor(int i, at::ScalarType type, int64_t dims) {
    if (!THPVariable_Check(v[i])) return fail();
    const at::Tensor& t = THPVariable_Unpack(v[i]);
    return t.scalar_type() == type && t.dim() == dims && t.get_device() == dev && !t.is_meta() ? &t : fail();
  }
  const at::Tensor* fail() {
    good = false;
    return nullptr;
  }
  // A contiguous tensor of these sizes (-1: any).
  void* dense(int i, at::ScalarType type, std::initializer_list<int64_t> sizes) {
    const at::Tensor* t = tensor(i, type, (int64_t)sizes.size());
    if (!t) return nullptr;
    int64_t d = 0;
    for (int64_t n : sizes) {
      if (n >= 0 && t->size(d) != n) return fail(), nullptr;
      ++d;
    }
    return t->is_contiguous() ? t->data_ptr() : (fail(), nullptr);
  }
  void* dense_or_none(int i, at::ScalarType type, std::initializer_list<int64_t> sizes) {
    return v[i] == Py_None ? nullptr : dense(i, type, sizes);
  }
  // bf16 [n, heads, D] with a dense last axis (n, heads -1: any).
  const at::Tensor* rows(int i, int64_t n, int64_t heads, int64_t D) {
    const at::Tensor* t = tensor(i, at::kBFloat16, 3);
    if (!t) return nullptr;
    const bool fits = (n < 0 || t->size(0) == n) && (heads < 0 || t->size(1) == heads) && t->size(2) == D &&
                      (t->stride(2) == 1 || t->numel() == 0);
    return fits ? t : fail();
  }
  template <typename T>
  T address(int i) {
    return reinterpret_cast<T>(PyLong_AsVoidPtr(v[i]));
  }
};

constexpr int64_t kMaxInt = 0x7FFFFFFF;
bool is_int(int64_t n) { return n <= kMaxInt; }

// An axis's stride; 0 where nothing is read at it (torch gives an axis of size 1 any stride, the entry
// points take multiples of 8).
int64_t step(const at::Tensor& t, int64_t axis) { return t.size(axis) > 1 ? t.stride(axis) : 0; }

PyObject* status(bool good, int rc) {
  if (PyErr_Occurred()) return nullptr;
  if (!good) Py_RETURN_NONE;
  return PyLong_FromLong(rc);
}

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const std::exception& e) {  // of torch, for a tensor without storage or strides
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

bool takes(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "expects %zd arguments, got %zd", want, n);
  return false;
}

// prep(entry, cache, device, rope, k, v, pages, at, seq, q, q_out, pos, q_norm, k_norm, eps, stream)
PyObject* prep(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  if (!takes(nargs, 16)) return nullptr;
  return guarded([&]() -> PyObject* {
    Args a{v};
    const auto entry = a.address<decltype(&qh_attn_prep_paged)>(0);
    const auto* cache = a.address<const qh_paged_cache*>(1);
    a.dev = (int)PyLong_AsLong(v[2]);
    const auto* rope = a.address<const qh_rope_axes*>(3);
    const float eps = (float)PyFloat_AsDouble(v[14]);
    void* stream = a.address<void*>(15);
    if (PyErr_Occurred()) return nullptr;
    const int64_t D = cache->head_dim, n_kv = cache->n_kv;
    const at::Tensor* k = a.rows(4, -1, n_kv, D);
    const int64_t T = k ? k->size(0) : 0;
    const at::Tensor* vv = a.rows(5, T, n_kv, D);
    if (k && vv && n_kv > 1 && T > 0) a.good = a.good && k->stride(1) == D && vv->stride(1) == D;
    const int* pages = (const int*)a.dense(6, at::kInt, {-1, -1});
    const int* where = (const int*)a.dense(7, at::kInt, {T});
    const int* seq = (const int*)a.dense_or_none(8, at::kInt, {T});
    const int* pos = nullptr;
    if (rope) {
      const int64_t axes = rope->n_axes;
      const bool flat = axes == 1 && THPVariable_Check(v[11]) && THPVariable_Unpack(v[11]).dim() == 1;
      pos = (const int*)(flat ? a.dense(11, at::kInt, {T}) : a.dense(11, at::kInt, {axes, T}));
    }
    const float* wq = (const float*)a.dense_or_none(12, at::kFloat, {D});
    const float* wk = (const float*)a.dense_or_none(13, at::kFloat, {D});
    const void* qp = nullptr;
    void* out = nullptr;
    int64_t H = 0, qs = 0, qh = 0;
    int f32 = 0;
    if (v[9] != Py_None) {
      if (const at::Tensor* q = a.rows(9, T, -1, D)) {
        H = q->size(1);
        qs = step(*q, 0);
        qh = step(*q, 1);
        qp = q->data_ptr();
        f32 = THPVariable_Check(v[10]) && THPVariable_Unpack(v[10]).scalar_type() == at::kFloat;
        out = a.dense(10, f32 ? at::kFloat : at::kBFloat16, {T, H, D});
      }
    } else if (v[10] != Py_None) {
      a.fail();
    }
    int rc = 0;
    if (a.good && is_int(T) && is_int(H)) {
      const at::Tensor& table = THPVariable_Unpack(v[6]);
      const int64_t n_seqs = table.size(0), max_pages = table.size(1);
      if (!is_int(n_seqs) || !is_int(max_pages)) Py_RETURN_NONE;
      const void *kp = k->data_ptr(), *vp = vv->data_ptr();
      const int64_t ks = step(*k, 0), vs = step(*vv, 0);
      Py_BEGIN_ALLOW_THREADS
      rc = entry(cache, rope, qp, qs, qh, kp, ks, vp, vs, wq, wk, eps, pos, seq, where, (int)T, pages, (int)n_seqs,
                 (int)max_pages, out, f32, (int)H, stream);
      Py_END_ALLOW_THREADS
    } else {
      a.good = false;
    }
    return status(a.good, rc);
  });
}

// read(entry, cache, device, pages, last, k_out, v_out, stream)
PyObject* read(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  if (!takes(nargs, 8)) return nullptr;
  return guarded([&]() -> PyObject* {
    Args a{v};
    const auto entry = a.address<decltype(&qh_kv_read_paged)>(0);
    const auto* cache = a.address<const qh_paged_cache*>(1);
    a.dev = (int)PyLong_AsLong(v[2]);
    void* stream = a.address<void*>(7);
    if (PyErr_Occurred()) return nullptr;
    const at::Tensor* table = a.tensor(3, at::kInt, 2);
    const int64_t B = table ? table->size(0) : 0, max_pages = table ? table->size(1) : 0;
    const int* pages = (const int*)a.dense(3, at::kInt, {-1, -1});
    const int* last = (const int*)a.dense(4, at::kInt, {B});
    const at::Tensor* k = a.tensor(5, at::kBFloat16, 4);
    const int64_t max_seq = k ? k->size(2) : 0;
    void* kp = a.dense(5, at::kBFloat16, {B, cache->n_kv, max_seq, cache->head_dim});
    void* vp = a.dense(6, at::kBFloat16, {B, cache->n_kv, max_seq, cache->head_dim});
    int rc = 0;
    a.good = a.good && is_int(B) && is_int(max_pages) && is_int(max_seq);
    if (a.good) {
      Py_BEGIN_ALLOW_THREADS
      rc = entry(cache, pages, (int)B, (int)max_pages, last, kp, vp, (int)max_seq, stream);
      Py_END_ALLOW_THREADS
    }
    return status(a.good, rc);
  });
}

// attend(entry, cache, device, q, pages, last, ws, gate, out, stream)
PyObject* attend(PyObject*, PyObject* const* v, Py_ssize_t nargs) {
  if (!takes(nargs, 10)) return nullptr;
  return guarded([&]() -> PyObject* {
    Args a{v};
    const auto entry = a.address<decltype(&qh_attn_decode_paged)>(0);
    const auto* cache = a.address<const qh_paged_cache*>(1);
    a.dev = (int)PyLong_AsLong(v[2]);
    void* stream = a.address<void*>(9);
    if (PyErr_Occurred()) return nullptr;
    const int64_t D = cache->head_dim;
    const at::Tensor* q = a.rows(3, -1, -1, D);
    const int64_t B = q ? q->size(0) : 0, H = q ? q->size(1) : 0;
    const int* pages = (const int*)a.dense(4, at::kInt, {B, -1});
    const int* last = (const int*)a.dense(5, at::kInt, {B});
    void* ws = a.dense(6, at::kByte, {-1});
    const at::Tensor* gate = v[7] == Py_None ? nullptr : a.rows(7, B, H, D);
    void* out = a.dense(8, at::kBFloat16, {B, H, D});
    int rc = 0;
    a.good = a.good && is_int(B) && is_int(H);
    if (a.good) {
      const int64_t max_pages = THPVariable_Unpack(v[4]).size(1), ws_bytes = THPVariable_Unpack(v[6]).size(0);
      if (!is_int(max_pages)) Py_RETURN_NONE;
      const void *qp = q->data_ptr(), *gp = gate ? gate->data_ptr() : nullptr;
      const int64_t qs = step(*q, 0), qh = step(*q, 1), gs = gate ? step(*gate, 0) : 0, gh = gate ? step(*gate, 1) : 0;
      Py_BEGIN_ALLOW_THREADS
      rc = entry(cache, qp, qs, qh, gp, gs, gh, pages, (int)B, (int)max_pages, last, (int)H, out, ws, (size_t)ws_bytes,
                 stream);
      Py_END_ALLOW_THREADS
    }
    return status(a.good, rc);
  });
}

PyMethodDef methods[] = {
    {"prep", (PyCFunction)(void (*)(void))prep, METH_FASTCALL, "Check the tensors of PagedKVCache.prep and launch it."},
    {"read", (PyCFunction)(void (*)(void))read, METH_FASTCALL, "Check the tensors of PagedKVCache.read and launch it."},
    {"attend", (PyCFunction)(void (*)(void))attend, METH_FASTCALL, "Check the tensors of PagedKVCache.attend and launch it."},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__paged_host() { return PyModule_Create(&module); }
