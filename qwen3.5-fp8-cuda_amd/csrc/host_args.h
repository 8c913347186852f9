// What the extension modules' functions share (paged_host.cpp, serve_host.cpp): the checks of a call's
// torch tensors, which note a misfit and hand back what the C entry point takes.
#pragma once

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <exception>

#include <torch/csrc/autograd/python_variable.h>

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
  // [n, width] with a dense last axis (n, width -1: any).
  const at::Tensor* matrix(int i, int64_t n, int64_t width, at::ScalarType type = at::kBFloat16) {
    const at::Tensor* t = tensor(i, type, 2);
    if (!t) return nullptr;
    const bool fits = (n < 0 || t->size(0) == n) && (width < 0 || t->size(1) == width) && (t->stride(1) == 1 || t->size(1) <= 1 || t->numel() == 0);
    return fits ? t : fail();
  }
  template <typename T>
  T address(int i) {
    return reinterpret_cast<T>(PyLong_AsVoidPtr(v[i]));
  }
};

constexpr int64_t kMaxInt = 0x7FFFFFFF;
inline bool is_int(int64_t n) { return n <= kMaxInt; }

// An axis's stride; 0 where nothing is read at it (torch gives an axis of size 1 any stride, the entry
// points take multiples of 8).
inline int64_t step(const at::Tensor& t, int64_t axis) { return t.size(axis) > 1 ? t.stride(axis) : 0; }

inline PyObject* status(bool good, int rc) {
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

inline bool takes(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "expects %zd arguments, got %zd", want, n);
  return false;
}

}  // namespace
